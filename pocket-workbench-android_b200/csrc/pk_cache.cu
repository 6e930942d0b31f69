// pk_cache.cu -- the quantised paged K/V cache: rows quantised as they are
// written, read back, and moved when drafts are accepted.  No counterpart in
// the reference, whose cache is f32 (model.rs:352-387).
//
// A row of head_dim values is held by head_dim / 8 lanes, 8 values each, so a
// warp has 2 (head_dim 128) or 4 (64) rows at once: 16-byte loads of half
// precision, 8- or 4-byte stores of codes, each row's bytes contiguous over
// its lanes.  The largest magnitude goes over the row's lanes by shuffles
// (Q4: over the four lanes of each 32 dimensions first).
#include "pk_cache.cuh"
#include "pk_cache.h"

namespace pk {
namespace {

constexpr int CT = 128;  // threads of a CTA

// round(x / d) to even for |x / d| < 2^20, exactly, with inv = 1 / d: the
// product x inv is within 3 f32 roundings of the quotient, which can only move
// a value across the middle between two codes; the remainder x - d c, exact in
// f32 (both terms are multiples of the smaller one's last place and the
// difference is below 2 d), tells on which side of it x lies.
__device__ __forceinline__ float code_of(float x, float d, float inv) {
  float c = rintf(isinf(inv) ? fdiv(x, d) : fmul(x, inv));  // (1 / d overflows for d < 2^-128)
  const float r = __fmaf_rn(-d, c, x), h = 0.5f * d, a = fabsf(r);
  if (a > h || (a == h && (((int)c) & 1))) c += r > 0.0f ? 1.0f : -1.0f;
  return c;
}

struct RowsArgs {
  pk_kv_cache c;
  pk_kv_seqs s;
  const void *src[2];
  void *dst[2];
  long tok_stride, head_stride;
  int vec, parts;
};

// A warp has one token and U sets of its rows (row r < 2 n_kv of a token is K,
// r < n_kv, or V of kv head r mod n_kv): the rows' values are asked for
// before the token's sequence, position and page are looked up, a chain of
// four dependent reads that is the same for all of them.
constexpr int U = 4;
struct Place {
  int t, set0, lane, l;
};
__device__ __forceinline__ Place place_of(int parts, int L) {
  const long long w = (long long)blockIdx.x * (CT / 32) + (threadIdx.x >> 5);
  Place p;
  p.t = (int)(w / parts);
  p.set0 = (int)(w - (long long)p.t * parts) * U;
  p.lane = threadIdx.x & 31;
  p.l = p.lane % L;
  return p;
}
// The cache row of kv head 0 at token t's position, or -1 (no sequence, past
// the bounds, no page); *mine: the token is some sequence's.
__device__ __forceinline__ long long head0_row(const RowsArgs &a, int t, int lane, bool *mine) {
  *mine = false;
  const int s = seq_of(a.s, t, lane);
  if (s < 0) return -1;
  const SeqView sv = seq_view(a.s, a.c.page_size, s);
  const int i = t - sv.first, p = sv.ctx + i;
  *mine = i < sv.n;
  if (i >= sv.n || sv.ctx < 0 || p >= sv.total) return -1;
  return row_at(a.c, a.s, s, p, 0);
}

template <int TYPE, int DH, int T>
__global__ void __launch_bounds__(CT) k_kv_store(const RowsArgs a) {
  using E = elem_t<T>;
  constexpr int L = DH / 8, RW = 32 / L;
  pdl_trigger();
  pdl_wait();
  const Place pl = place_of(a.parts, L);
  if (pl.t >= a.s.n_tok) return;
  const int l = pl.l, lane = pl.lane;
  float x[U][8];
#pragma unroll
  for (int k = 0; k < U; k++) {
    const int r = (pl.set0 + k) * RW + lane / L, which = r >= a.c.n_kv ? 1 : 0;
    if (r < 2 * a.c.n_kv) {
      load_n<E, 8>(reinterpret_cast<const E *>(which ? a.src[1] : a.src[0]) + (long long)pl.t * a.tok_stride +
                       (long long)(r - which * a.c.n_kv) * a.head_stride + 8 * l,
                   a.vec, x[k]);
    } else {
#pragma unroll
      for (int i = 0; i < 8; i++) x[k][i] = 0.0f;
    }
  }
  bool mine;
  const long long row0 = head0_row(a, pl.t, lane, &mine);
  if (row0 < 0) return;
#pragma unroll
  for (int k = 0; k < U; k++) {
    const int r = (pl.set0 + k) * RW + lane / L, which = r >= a.c.n_kv ? 1 : 0;
    const bool on = r < 2 * a.c.n_kv;
    if ((pl.set0 + k) * RW >= 2 * a.c.n_kv) break;  // (the whole warp)
    const size_t row = (size_t)row0 + (size_t)(r - which * a.c.n_kv) * a.c.page_size;
    float m = 0.0f;
#pragma unroll
    for (int i = 0; i < 8; i++) {
      x[k][i] = isnan(x[k][i]) ? 0.0f : fminf(fmaxf(x[k][i], -0x1p127f), 0x1p127f);
      m = fmaxf(m, fabsf(x[k][i]));
    }
    uint8_t *codes = reinterpret_cast<uint8_t *>(which ? a.c.v : a.c.k);
    float *scales = which ? a.c.vs : a.c.ks;
    if (TYPE == PK_KV_Q8) {
#pragma unroll
      for (int o = L / 2; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
      const float d = fdiv(m, 127.0f), inv = fdiv(1.0f, d);
      uint32_t u[2] = {0, 0};
#pragma unroll
      for (int i = 0; i < 8; i++) {
        const float c = d > 0.0f ? fminf(fmaxf(code_of(x[k][i], d, inv), -127.0f), 127.0f) : 0.0f;
        u[i / 4] |= (uint32_t)((int)c + 128) << (8 * (i % 4));
      }
      if (on) {
        *reinterpret_cast<uint2 *>(codes + row * DH + 8 * l) = make_uint2(u[0], u[1]);
        if (l == 0) scales[row] = d;
      }
    } else {
#pragma unroll
      for (int o = 2; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
      const float mb = m;  // of the 32 dimensions
#pragma unroll
      for (int o = L / 2; o > 2; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
      const float d = fdiv(m, 105.0f);
      // d == 0: the quotient is NaN (0 / 0) or infinite, and the row stands for 0 either way
      const float sb = d > 0.0f ? fminf(fmaxf(ceilf(fdiv(mb, fmul(7.0f, d))), 1.0f), 15.0f) : 1.0f;
      const float step = fmul(d, sb), inv = fdiv(1.0f, step);
      uint32_t u = 0;
#pragma unroll
      for (int i = 0; i < 8; i++) {
        const float c = step > 0.0f ? fminf(fmaxf(code_of(x[k][i], step, inv), -8.0f), 7.0f) : 0.0f;
        u |= (uint32_t)((int)c + 8) << (4 * i);
      }
      uint32_t word = 0;
#pragma unroll
      for (int b = 0; b < DH / 32; b++) word |= (uint32_t)__shfl_sync(0xffffffffu, sb, lane - l + 4 * b) << (4 * b);
      if (on) {
        *reinterpret_cast<uint32_t *>(codes + row * (DH / 2) + 4 * l) = u;
        if (l == 0) *reinterpret_cast<float2 *>(scales + 2 * row) = make_float2(d, __uint_as_float(word));
      }
    }
  }
}

template <int TYPE, int DH, int T>
__global__ void __launch_bounds__(CT) k_kv_load(const RowsArgs a) {
  using E = elem_t<T>;
  constexpr int L = DH / 8, RW = 32 / L;
  pdl_trigger();
  pdl_wait();
  const Place pl = place_of(a.parts, L);
  if (pl.t >= a.s.n_tok) return;
  const int l = pl.l;
  bool mine;
  const long long row0 = head0_row(a, pl.t, pl.lane, &mine);
  if (!mine) return;
  uint2 u[U];
  float2 d[U];
#pragma unroll
  for (int k = 0; k < U; k++) {
    const int r = (pl.set0 + k) * RW + pl.lane / L, which = r >= a.c.n_kv ? 1 : 0;
    u[k] = make_uint2(0, 0);
    d[k] = make_float2(0.0f, 0.0f);  // no page: D = 0
    if (row0 < 0 || r >= 2 * a.c.n_kv) continue;
    const size_t row = (size_t)row0 + (size_t)(r - which * a.c.n_kv) * a.c.page_size;
    const uint8_t *codes = reinterpret_cast<const uint8_t *>(which ? a.c.v : a.c.k);
    const float *scales = which ? a.c.vs : a.c.ks;
    if (TYPE == PK_KV_Q8) {
      u[k] = *reinterpret_cast<const uint2 *>(codes + row * DH + 8 * l);
      d[k].x = scales[row];
    } else {
      u[k].x = *reinterpret_cast<const uint32_t *>(codes + row * (DH / 2) + 4 * l);
      d[k] = *reinterpret_cast<const float2 *>(scales + 2 * row);
    }
  }
#pragma unroll
  for (int k = 0; k < U; k++) {
    const int r = (pl.set0 + k) * RW + pl.lane / L, which = r >= a.c.n_kv ? 1 : 0;
    if (r >= 2 * a.c.n_kv) continue;
    float x[8];
    if (TYPE == PK_KV_Q8) {
#pragma unroll
      for (int i = 0; i < 8; i++) x[i] = fmul(d[k].x, (float)((int)(((i < 4 ? u[k].x : u[k].y) >> (8 * (i % 4))) & 255u) - 128));
    } else {
      const int sb = (int)((__float_as_uint(d[k].y) >> (4 * (l / 4))) & 15u);
#pragma unroll
      for (int i = 0; i < 8; i++) x[i] = fmul(d[k].x, (float)(((int)((u[k].x >> (4 * i)) & 15u) - 8) * sb));
    }
    if (row0 < 0) {
#pragma unroll
      for (int i = 0; i < 8; i++) x[i] = 0.0f;
    }
    store_n<E, 8>(reinterpret_cast<E *>(which ? a.dst[1] : a.dst[0]) + (long long)pl.t * a.tok_stride +
                      (long long)(r - which * a.c.n_kv) * a.head_stride + 8 * l,
                  a.vec, x);
  }
}

// Accepted drafts: a warp owns (sequence, kv head, K or V) and moves its rows
// in batches of KB, reading a batch before it writes it.  keep[j] >= j, so a
// row written (at most j) is never one that a later batch still reads.
constexpr int KB = 8;
template <int TYPE, int DH>
__global__ void __launch_bounds__(CT) k_kv_keep(const pk_kv_cache c, const pk_kv_seqs q, const int *keep,
                                                int keep_stride, const int *n_keep) {
  constexpr int RB = TYPE == PK_KV_Q8 ? DH : DH / 2, SW = TYPE == PK_KV_Q8 ? 1 : 2;
  constexpr int L = RB / 16;        // lanes of a row's codes, 16 bytes each
  constexpr int RP = 32 / L;        // rows a pass
  constexpr int P = (KB + RP - 1) / RP;
  pdl_trigger();
  pdl_wait();
  const int lane = threadIdx.x & 31;
  const long long w = (long long)blockIdx.x * (CT / 32) + (threadIdx.x >> 5);
  const int per = 2 * c.n_kv;
  if (w >= (long long)q.n_seq * per) return;
  const int s = (int)(w / per), r = (int)(w - (long long)s * per), which = r >= c.n_kv ? 1 : 0, h = r - which * c.n_kv;
  const SeqView sv = seq_view(q, c.page_size, s);
  if (sv.ctx < 0) return;
  const int n = min(min(__ldg(n_keep + s), keep_stride), sv.n);
  uint8_t *codes = reinterpret_cast<uint8_t *>(which ? c.v : c.k);
  float *scales = which ? c.vs : c.ks;
  for (int j0 = 0; j0 < n; j0 += RP * P) {
    uint4 u[P];
    float sc[P][SW];
    long long to[P];
#pragma unroll
    for (int i = 0; i < P; i++) {
      const int j = j0 + i * RP + lane / L;
      to[i] = -1;
      if (j >= n) continue;
      const int from = __ldg(keep + (size_t)s * keep_stride + j);
      if (from < j || from >= sv.n || from == j || sv.ctx + from >= sv.total) continue;
      const long long src = row_at(c, q, s, sv.ctx + from, h);
      if (src < 0) continue;
      to[i] = row_at(c, q, s, sv.ctx + j, h);
      u[i] = *reinterpret_cast<const uint4 *>(codes + (size_t)src * RB + 16 * (lane % L));
#pragma unroll
      for (int e = 0; e < SW; e++) sc[i][e] = scales[src * SW + e];
    }
    __syncwarp();
#pragma unroll
    for (int i = 0; i < P; i++) {
      if (to[i] < 0) continue;
      *reinterpret_cast<uint4 *>(codes + (size_t)to[i] * RB + 16 * (lane % L)) = u[i];
      if (lane % L == 0) {
#pragma unroll
        for (int e = 0; e < SW; e++) scales[to[i] * SW + e] = sc[i][e];
      }
    }
    __syncwarp();
  }
}

template <class... KArgs, class... Args>
cudaError_t launch(void (*kernel)(KArgs...), dim3 grid, dim3 block, size_t smem, cudaStream_t st, Args... args) {
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = grid;
  cfg.blockDim = block;
  cfg.dynamicSmemBytes = smem;
  cfg.stream = st;
  cudaLaunchAttribute at{};
  at.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  at.val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = &at;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, kernel, static_cast<KArgs>(args)...);
}

template <int TYPE, int DH>
cudaError_t rows_launch(bool store, const RowsArgs &a, int type, dim3 grid, cudaStream_t st) {
  void (*k)(RowsArgs) = nullptr;
  if (store) k = type == T_F32 ? k_kv_store<TYPE, DH, T_F32> : type == T_F16 ? k_kv_store<TYPE, DH, T_F16> : k_kv_store<TYPE, DH, T_BF16>;
  else k = type == T_F32 ? k_kv_load<TYPE, DH, T_F32> : type == T_F16 ? k_kv_load<TYPE, DH, T_F16> : k_kv_load<TYPE, DH, T_BF16>;
  return launch(k, grid, dim3(CT), 0, st, a);
}

cudaError_t rows(bool store, RowsArgs a, int type, cudaStream_t st) {
  const size_t es = type == T_F32 ? 4 : 2;
  const uintptr_t p0 = (uintptr_t)(store ? a.src[0] : a.dst[0]), p1 = (uintptr_t)(store ? a.src[1] : a.dst[1]);
  a.vec = ((p0 | p1 | (uintptr_t)(a.tok_stride * (long)es) | (uintptr_t)(a.head_stride * (long)es)) & 15) == 0;
  const int rw = 32 / (a.c.head_dim / 8);
  a.parts = (2 * a.c.n_kv + rw * U - 1) / (rw * U);
  const long long warps = (long long)a.s.n_tok * a.parts, blocks = (warps + CT / 32 - 1) / (CT / 32);
  if (blocks > 0x7fffffffLL) return cudaErrorInvalidValue;
  const dim3 grid((unsigned)blocks);
  if (a.c.type == PK_KV_Q8)
    return a.c.head_dim == 64 ? rows_launch<PK_KV_Q8, 64>(store, a, type, grid, st)
                              : rows_launch<PK_KV_Q8, 128>(store, a, type, grid, st);
  return a.c.head_dim == 64 ? rows_launch<PK_KV_Q4, 64>(store, a, type, grid, st)
                            : rows_launch<PK_KV_Q4, 128>(store, a, type, grid, st);
}

}  // namespace

cudaError_t launch_kv_store(const pk_kv_cache &c, const pk_kv_seqs &s, const void *k, const void *v, int type,
                            long tok_stride, long head_stride, cudaStream_t st) {
  RowsArgs a{};
  a.c = c; a.s = s;
  a.src[0] = k; a.src[1] = v;
  a.tok_stride = tok_stride; a.head_stride = head_stride;
  return rows(true, a, type, st);
}

cudaError_t launch_kv_load(const pk_kv_cache &c, const pk_kv_seqs &s, void *k, void *v, int type, long tok_stride,
                           long head_stride, cudaStream_t st) {
  RowsArgs a{};
  a.c = c; a.s = s;
  a.dst[0] = k; a.dst[1] = v;
  a.tok_stride = tok_stride; a.head_stride = head_stride;
  return rows(false, a, type, st);
}

cudaError_t launch_kv_keep(const pk_kv_cache &c, const pk_kv_seqs &s, const int *keep, int keep_stride,
                           const int *n_keep, cudaStream_t st) {
  const long long warps = (long long)s.n_seq * 2 * c.n_kv, blocks = (warps + CT / 32 - 1) / (CT / 32);
  if (blocks > 0x7fffffffLL) return cudaErrorInvalidValue;
  void (*k)(pk_kv_cache, pk_kv_seqs, const int *, int, const int *) =
      c.type == PK_KV_Q8 ? (c.head_dim == 64 ? k_kv_keep<PK_KV_Q8, 64> : k_kv_keep<PK_KV_Q8, 128>)
                         : (c.head_dim == 64 ? k_kv_keep<PK_KV_Q4, 64> : k_kv_keep<PK_KV_Q4, 128>);
  return launch(k, dim3((unsigned)blocks), dim3(CT), 0, st, c, s, keep, keep_stride, n_keep);
}

}  // namespace pk
