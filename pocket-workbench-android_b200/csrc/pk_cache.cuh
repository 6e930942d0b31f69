// pk_cache.cuh -- device helpers of the quantised paged cache's kernels.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <stdint.h>

#include "pk.h"
#include "pk_device.cuh"

namespace pk {

// Element types of the op-level tensors.
template <int T> struct Elem;
template <> struct Elem<T_F32> { using type = float; };
template <> struct Elem<T_F16> { using type = __half; };
template <> struct Elem<T_BF16> { using type = __nv_bfloat16; };
template <int T> using elem_t = typename Elem<T>::type;
__device__ __forceinline__ float to_f(float v) { return v; }
__device__ __forceinline__ float to_f(__half v) { return __half2float(v); }
__device__ __forceinline__ float to_f(__nv_bfloat16 v) { return __bfloat162float(v); }
template <class E> __device__ __forceinline__ E from_f(float v);
template <> __device__ __forceinline__ float from_f<float>(float v) { return v; }
template <> __device__ __forceinline__ __half from_f<__half>(float v) { return __float2half_rn(v); }
template <> __device__ __forceinline__ __nv_bfloat16 from_f<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }

// N consecutive elements as f32 and back; vec: p is aligned to 16 bytes.
template <class E, int N>
__device__ __forceinline__ void load_n(const E *p, bool vec, float (&v)[N]) {
  constexpr int B = N * (int)sizeof(E);
  static_assert(B % 16 == 0, "whole 16-byte words");
  if (vec) {
    uint4 w[B / 16];
#pragma unroll
    for (int i = 0; i < B / 16; i++) w[i] = __ldg(reinterpret_cast<const uint4 *>(p) + i);
    const E *e = reinterpret_cast<const E *>(w);
#pragma unroll
    for (int i = 0; i < N; i++) v[i] = to_f(e[i]);
  } else {
#pragma unroll
    for (int i = 0; i < N; i++) v[i] = to_f(p[i]);
  }
}
template <class E, int N>
__device__ __forceinline__ void store_n(E *p, bool vec, const float (&v)[N]) {
  constexpr int B = N * (int)sizeof(E);
  static_assert(B % 16 == 0, "whole 16-byte words");
  if (vec) {
    uint4 w[B / 16];
    E *e = reinterpret_cast<E *>(w);
#pragma unroll
    for (int i = 0; i < N; i++) e[i] = from_f<E>(v[i]);
#pragma unroll
    for (int i = 0; i < B / 16; i++) reinterpret_cast<uint4 *>(p)[i] = w[i];
  } else {
#pragma unroll
    for (int i = 0; i < N; i++) p[i] = from_f<E>(v[i]);
  }
}

__device__ __forceinline__ uint32_t h2u(__half2 h) { return *reinterpret_cast<uint32_t *>(&h); }
__device__ __forceinline__ __half2 u2h(uint32_t u) { return *reinterpret_cast<__half2 *>(&u); }

// Bytes x_i = c_i + 128 in the low and high halves of (1024 + x) f16 words:
// 0x6400 | x is 1024 + x, and 1152 taken off leaves c exactly.
__device__ __forceinline__ uint32_t codes_of(uint32_t bytes, uint32_t sel) {
  return h2u(__hsub2(u2h(__byte_perm(bytes, 0x64646464u, sel)), u2h(0x64806480u)));
}
// Nibbles x = c + 8 at bits 0-3 and 16-19: (1024 + x) s - 1032 s = c s, exact.
__device__ __forceinline__ uint32_t nibbles_of(uint32_t w, uint32_t s, uint32_t m1032s) {
  return h2u(__hfma2(u2h((w & 0x000f000fu) | 0x64006400u), u2h(s), u2h(m1032s)));
}
__device__ __forceinline__ uint32_t dup_h(int s) { return h2u(__half2half2(__int2half_rn(s))); }

// One sequence's bounds, made safe whatever the device arrays hold: rows
// [first, first + n) of the token arrays, n <= max_new; total = positions in
// reach, at most max_len and what the page table addresses (none for a
// negative ctx); committed positions ctx, at most as many (what is past them
// is out of reach anyway, and sums with a larger one could wrap).
struct SeqView {
  int first, n, ctx, total;
};
__device__ __forceinline__ SeqView seq_view(const pk_kv_seqs &q, int page_size, int s) {
  SeqView v;
  const int a = __ldg(q.start + s), b = __ldg(q.start + s + 1), c = __ldg(q.ctx + s);
  v.first = min(max(a, 0), q.n_tok);
  v.n = min(max(min(b, q.n_tok) - v.first, 0), q.max_new);
  const long long cap = min((long long)q.max_pages * page_size, (long long)q.max_len);
  v.ctx = (int)min((long long)c, cap);
  v.total = c < 0 ? 0 : (int)min((long long)c + v.n, cap);
  return v;
}
// The last i < n with at[i] <= t, by a whole warp: 32 probes a level.  -1 when
// t lies before the first.
__device__ __forceinline__ int last_at(const int *at, int n, int t, int lane) {
  int lo = 0, len = n;  // at[lo .. lo + len) holds the answer
  while (len > 1) {
    const int step = (len + 31) / 32, i = lo + lane * step;
    const bool le = lane * step < len && __ldg(at + i) <= t;
    const int n = __popc(__ballot_sync(0xffffffffu, le));
    if (n == 0) return -1;
    const int adv = (n - 1) * step;
    lo += adv;
    len = min(step, len - adv);
  }
  return __ldg(at + lo) <= t ? lo : -1;
}
// The sequence that token row t belongs to (the last s with start[s] <= t).
__device__ __forceinline__ int seq_of(const pk_kv_seqs &q, int t, int lane) { return last_at(q.start, q.n_seq, t, lane); }
// Index of the cache row of (position p, kv head h), or -1 where there is no page.
__device__ __forceinline__ long long row_at(const pk_kv_cache &c, const pk_kv_seqs &q, int s, int p, int h) {
  const int j = p / c.page_size;
  if (p < 0 || j >= q.max_pages) return -1;
  const int page = __ldg(q.pages + (size_t)s * q.max_pages + j);
  if (page < 0 || page >= c.n_pages) return -1;
  return ((long long)page * c.n_kv + h) * c.page_size + (p - j * c.page_size);
}

}  // namespace pk
