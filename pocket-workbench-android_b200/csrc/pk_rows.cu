// pk_rows.cu -- kernels that go over rows once: rotary positions and the
// rules on logits.  The engine's own RoPE (k_rope_kv, model.rs:408-461) reads
// f32 tables of every position; these are the op level's, for any position.
#include <math_constants.h>

#include <algorithm>

#include "pk_cache.cuh"
#include "pk_cache.h"
#include "pk_launch.h"

namespace pk {
namespace {

// ------------------------------------------------------------------- rotary
// A CTA takes one token and some of its heads: the angles once for them all
// (double: position times turns, less its whole turns, is exact to 2^-53 of
// the angle; the remainder, at most half a turn, is rounded to f32 for its
// cosine and sine, 2^-26 of a turn or 9.4e-8 of the pair's length at the most:
// f32 outputs are 6.5e-8 from 64 bits, 4.6e-8 with double ones), while the first values
// are on their way.  An item is V elements (16 bytes where everything is
// aligned for it): for interleaved pairs a run of a head's dimensions, for
// the half layout V pairs' two runs, or a run that is copied.  A thread keeps
// its place in the head and goes from head to head, so its cosines and sines
// stay in registers and its addresses are additions (with an item's place
// divided out anew, index arithmetic was half the kernel's instructions).
// 8191 tokens of 72 heads of 64, 48 rotated, f16: 34 us, 69% of a copy's rate.
constexpr int RT = 256;
// AL: whole runs, aligned to their size; otherwise moved by elements, the last
// run of an odd head_dim one short (n < V).
template <int V, bool AL, class X>
__device__ __forceinline__ void move_run(X *dst, const X *src, int n) {
  constexpr int B = V * (int)sizeof(X);
  if (AL && B == 16) *reinterpret_cast<uint4 *>(dst) = *reinterpret_cast<const uint4 *>(src);
  else if (AL && B == 8) *reinterpret_cast<uint2 *>(dst) = *reinterpret_cast<const uint2 *>(src);
  else if (AL && B == 4) *reinterpret_cast<uint32_t *>(dst) = *reinterpret_cast<const uint32_t *>(src);
  else
#pragma unroll
    for (int e = 0; e < V; e++)
      if (AL || e < n) dst[e] = src[e];
}

template <int T, int V, bool HALF, bool AL>
__global__ void __launch_bounds__(RT) k_rope(const pk_rope_args p, int heads_cta) {
  using E = elem_t<T>;
  constexpr int N = HALF ? 2 : 3;  // items in flight a thread
  constexpr int NP = HALF ? V : V / 2;  // pairs of an item
  extern __shared__ float2 cs[];  // [n_rot / 2]
  pdl_trigger();
  pdl_wait();
  const long long t = blockIdx.x;
  const int half = p.n_rot / 2, nq = p.q ? p.n_head : 0, heads = nq + (p.k ? p.n_kv : 0);
  // items a head: dimensions (interleaved), or pairs and the dimensions past them
  const int per = HALF ? (p.head_dim - half) / V : (p.head_dim + V - 1) / V;
  const int h1 = min(heads, ((int)blockIdx.y + 1) * heads_cta);
  const int wide = min(per, RT), step = RT / wide;  // threads a head, heads at a time
  const int row = (int)threadIdx.x / wide;
  const E *in[2] = {reinterpret_cast<const E *>(p.q) + t * p.q_tok_stride,
                    reinterpret_cast<const E *>(p.k) + t * p.k_tok_stride - nq * p.k_head_stride};
  E *out[2] = {reinterpret_cast<E *>(p.q_out) + t * p.qo_tok_stride,
               reinterpret_cast<E *>(p.k_out) + t * p.ko_tok_stride - nq * p.ko_head_stride};
  bool first = true;
  for (int k = (int)threadIdx.x - row * wide; first || k < per; k += wide) {
    const bool mine = row < step && k < per;
    const bool rot = HALF ? k * V < half : true;
    const int d = HALF && !rot ? k * V + half : k * V;  // past the pairs: dimensions n_rot ..
    const int len = HALF ? V : min(V, p.head_dim - d);
    float2 c[NP];
    for (int h = (int)blockIdx.y * heads_cta + row; first || h < h1; h += step * N) {
      alignas(16) E a[N][V], b[N][HALF ? V : 1];
#pragma unroll
      for (int n = 0; n < N; n++) {
        const int hh = h + n * step;
        if (!mine || hh >= h1) continue;
        const E *x = (hh >= nq ? in[1] + hh * p.k_head_stride : in[0] + hh * p.q_head_stride) + d;
        move_run<V, AL>(a[n], x, len);
        if (HALF && rot) move_run<V, AL>(b[n], x + half, len);
      }
      if (first) {
        first = false;
        const double pos = (double)__ldg(p.pos + t);
        for (int i = threadIdx.x; i < half; i += RT) {
          double r = pos * __ldg(p.turns + i);
          r -= rint(r);
          float sn, co;
          sincospif(2.0f * (float)r, &sn, &co);
          cs[i] = make_float2(co * p.gain, sn * p.gain);
        }
        __syncthreads();
      }
      if (!mine) break;
      if (h < (int)blockIdx.y * heads_cta + step) {
#pragma unroll
        for (int e = 0; e < NP; e++) {
          const int i = HALF ? k * V + e : k * V / 2 + e;
          c[e] = i < half ? cs[i] : make_float2(1.0f, 0.0f);
        }
      }
#pragma unroll
      for (int n = 0; n < N; n++) {
        const int hh = h + n * step;
        if (hh >= h1) continue;
        E *y = (hh >= nq ? out[1] + hh * p.ko_head_stride : out[0] + hh * p.qo_head_stride) + d;
        if (HALF) {
          if (rot) {
#pragma unroll
            for (int e = 0; e < V; e++) {
              const float u = to_f(a[n][e]), v = to_f(b[n][e]);
              a[n][e] = from_f<E>(u * c[e].x - v * c[e].y);
              b[n][e] = from_f<E>(u * c[e].y + v * c[e].x);
            }
            move_run<V, AL>(y + half, b[n], len);
          }
        } else {
#pragma unroll
          for (int e = 0; e + 1 < V; e += 2) {
            if (k * V / 2 + e / 2 >= half) break;  // past the pairs: copied as they are
            const float u = to_f(a[n][e]), v = to_f(a[n][e + 1]);
            a[n][e] = from_f<E>(u * c[e / 2].x - v * c[e / 2].y);
            a[n][e + 1] = from_f<E>(u * c[e / 2].y + v * c[e / 2].x);
          }
        }
        move_run<V, AL>(y, a[n], len);
      }
    }
  }
}

template <int T, int V, bool HALF, bool AL>
cudaError_t rope_as(const pk_rope_args &a, cudaStream_t st) {
  // few tokens: a token's heads over several CTAs, so that all SMs take part
  const int heads = (a.q ? a.n_head : 0) + (a.k ? a.n_kv : 0);
  const int want = std::max(1, std::min(heads, 592 / std::max(a.n_tok, 1)));
  const int per = (heads + want - 1) / want;
  return launch(k_rope<T, V, HALF, AL>, dim3((unsigned)a.n_tok, (unsigned)((heads + per - 1) / per)), dim3(RT),
                (int)(a.n_rot / 2 * sizeof(float2)), st, a, per);
}
template <int T>
cudaError_t rope_type(const pk_rope_args &a, cudaStream_t st) {
  constexpr int W = 16 / (int)sizeof(elem_t<T>);
  const bool half = a.layout == PK_ROPE_HALF;
  // whether items of V elements are whole and aligned
  auto fits = [&](int v) {
    uintptr_t bits = 0;
    if (a.q) bits |= (uintptr_t)a.q | (uintptr_t)a.q_out | ((uintptr_t)(a.q_tok_stride | a.q_head_stride | a.qo_tok_stride | a.qo_head_stride) * sizeof(elem_t<T>));
    if (a.k) bits |= (uintptr_t)a.k | (uintptr_t)a.k_out | ((uintptr_t)(a.k_tok_stride | a.k_head_stride | a.ko_tok_stride | a.ko_head_stride) * sizeof(elem_t<T>));
    return bits % (v * sizeof(elem_t<T>)) == 0 && a.head_dim % v == 0 && (!half || (a.n_rot / 2) % v == 0);
  };
  if (half) return fits(W) ? rope_as<T, W, true, true>(a, st) : fits(2) ? rope_as<T, 2, true, true>(a, st) : rope_as<T, 1, true, false>(a, st);
  return fits(W) ? rope_as<T, W, false, true>(a, st) : rope_as<T, 2, false, false>(a, st);
}

// -------------------------------------------------------------- logit rules
// Long lists: a CTA takes SEG logits of a row, NT threads.  All that it reads (logits,
// masks, the first HB NT history ids, the first NT biases, the row's numbers)
// is asked for at the start, while its counts are cleared, so that it waits
// for memory once.  It counts the row's ids that fall into its segment in
// shared memory (whole counts: their order does not matter) and collects the
// biases of the segment there, in the list's order, which one warp adds up.
// Then each token that was seen or biased is finished by the one thread that
// claims its count, and the segment goes out with those in their places:
// where every run of logits looked for its own, some lane of nearly every
// warp had one and all went through the division (91 us for 250 rows of
// 128256).
template <int T, int SEG, int NT, int CTAS>
__global__ void __launch_bounds__(NT, CTAS) k_logit_rules(const void *in, void *out, int n, long in_stride, long out_stride,
                                                          const pk_logit_rules r, int segs, int vec) {
  using E = elem_t<T>;
  constexpr int V = 16 / (int)sizeof(E), RUNS = SEG / (NT * V);  // a thread has runs of V elements
  constexpr int HB = 4, BIASED = 1 << 30;
  static_assert(RUNS * NT * V == SEG, "whole runs");
  extern __shared__ __align__(16) uint8_t smem[];
  int *cnt = reinterpret_cast<int *>(smem);                 // [SEG] counts; BIASED; -1: claimed
  float *val = reinterpret_cast<float *>(smem) + SEG;       // [SEG] biases, then finished values
  __shared__ uint32_t bid[NT];
  __shared__ float bval[NT];
  __shared__ int bcount[NT / 32];
  pdl_trigger();
  pdl_wait();
  const int row = blockIdx.x / segs;
  const int lo = (int)(blockIdx.x - row * segs) * SEG, m = min(SEG, n - lo), tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const E *x = reinterpret_cast<const E *>(in) + row * in_stride + lo;
  E *y = reinterpret_cast<E *>(out) + row * out_stride + lo;
  const uint32_t *ids = r.hist + row * r.hist_stride;
  const uint32_t *allow = r.allow ? r.allow + row * r.allow_stride + (lo >> 5) : nullptr;
  const bool touch = r.hist || r.bias_id;
  alignas(16) E v[RUNS][V];
  uint32_t ok[RUNS], hid[HB];
#pragma unroll
  for (int h = 0; h < HB; h++) hid[h] = 0xffffffffu;
#pragma unroll
  for (int k = 0; k < RUNS; k++) {
    const int i = (k * NT + tid) * V;
    ok[k] = 0xffffffffu;
    if (i >= m) continue;
    if (vec && i + V <= m) {
      *reinterpret_cast<uint4 *>(v[k]) = *reinterpret_cast<const uint4 *>(x + i);
    } else {
#pragma unroll
      for (int e = 0; e < V; e++)
        if (i + e < m) v[k][e] = x[i + e];
    }
    if (allow) ok[k] = __ldg(allow + (i >> 5)) >> (i & 31);  // V divides 32
  }
  int nh = 0;
  if (r.hist) {
    nh = r.n_hist ? __ldg(r.n_hist + row) : r.n_hist_max;
#pragma unroll
    for (int h = 0; h < HB; h++) {
      if (h * NT + tid < r.n_hist_max) hid[h] = __ldg(ids + h * NT + tid);
    }
  }
  uint32_t b_id = 0xffffffffu;
  float b_val = 0.0f;
  if (r.bias_id && tid < r.n_bias) {
    b_id = __ldg(r.bias_id + row * r.bias_stride + tid);
    b_val = __ldg(r.bias + row * r.bias_stride + tid);
  }
  if (touch) {
    for (int i = tid; i < (r.bias_id ? 2 : 1) * SEG / 4; i += NT) reinterpret_cast<uint4 *>(smem)[i] = make_uint4(0, 0, 0, 0);
    __syncthreads();
  }
  // the segment's place of history entry i (id: as read above), m or more: none
  auto place = [&](int i, uint32_t id) { return i < nh ? id - (uint32_t)lo : 0xffffffffu; };
  if (r.hist) {
    nh = min(max(nh, 0), r.n_hist_max);
#pragma unroll
    for (int h = 0; h < HB; h++) {
      const uint32_t d = place(h * NT + tid, hid[h]);
      if (d < (uint32_t)m) atomicAdd(&cnt[d], 1);
    }
    for (int i = HB * NT + tid; i < nh; i += NT) {
      const uint32_t d = place(i, __ldg(ids + i));
      if (d < (uint32_t)m) atomicAdd(&cnt[d], 1);
    }
  }
  if (r.bias_id) {
    for (int i0 = 0; i0 < r.n_bias; i0 += NT) {  // (uniform)
      uint32_t id = b_id;
      float b = b_val;
      if (i0 > 0) {
        id = i0 + tid < r.n_bias ? __ldg(r.bias_id + row * r.bias_stride + i0 + tid) : 0xffffffffu;
        b = i0 + tid < r.n_bias ? __ldg(r.bias + row * r.bias_stride + i0 + tid) : 0.0f;
      }
      const uint32_t d = i0 + tid < r.n_bias ? id - (uint32_t)lo : 0xffffffffu;
      const unsigned here = __ballot_sync(0xffffffffu, d < (uint32_t)m);
      if (lane == 0) bcount[warp] = __popc(here);
      __syncthreads();
      int at = __popc(here & ((1u << lane) - 1)), all = 0;
#pragma unroll
      for (int w = 0; w < NT / 32; w++) {
        at += w < warp ? bcount[w] : 0;
        all += bcount[w];
      }
      if (d < (uint32_t)m) {
        bid[at] = d;
        bval[at] = b;
        atomicOr(&cnt[d], BIASED);
      }
      __syncthreads();
      if (warp == 0) {
        for (int j0 = 0; j0 < all; j0 += 32) {
          const uint32_t at1 = j0 + lane < all ? bid[j0 + lane] : 0xffffffffu;
          const unsigned same = __match_any_sync(0xffffffffu, at1);
          if (at1 != 0xffffffffu) {
            for (unsigned left = same; left; left &= left - 1) {  // lanes with the same id, in order
              if (lane == __ffs(left) - 1) val[at1] += bval[j0 + lane];
              __syncwarp(same);
            }
          }
          __syncwarp();
        }
      }
      __syncthreads();
    }
  }
  if (touch) {
    const float rep = r.repeat ? __ldg(r.repeat + row) : 1.0f, fr = r.freq ? __ldg(r.freq + row) : 0.0f,
                pr = r.presence ? __ldg(r.presence + row) : 0.0f;
    __syncthreads();
    // claims the places d, all counts before all logits (each is a wait)
    auto claim = [&](auto &d) {
      constexpr int N = sizeof(d) / sizeof(d[0]);
      int c[N];
      float f[N];
#pragma unroll
      for (int i = 0; i < N; i++) c[i] = d[i] < (uint32_t)m ? atomicExch(&cnt[d[i]], -1) : 0;
#pragma unroll
      for (int i = 0; i < N; i++) f[i] = c[i] > 0 ? to_f(x[d[i]]) : 0.0f;
#pragma unroll
      for (int i = 0; i < N; i++) {
        if (c[i] <= 0) continue;  // (none, or claimed already)
        const int times = c[i] & (BIASED - 1);
        if (times > 0) {
          f[i] = f[i] > 0.0f ? fdiv(f[i], rep) : fmul(f[i], rep);
          f[i] = fsub(f[i], fadd(fmul((float)times, fr), pr));
        }
        val[d[i]] = c[i] & BIASED ? fadd(f[i], val[d[i]]) : f[i];
      }
    };
    uint32_t d[HB + 1];
#pragma unroll
    for (int h = 0; h < HB; h++) d[h] = place(h * NT + tid, hid[h]);
    d[HB] = r.bias_id && tid < r.n_bias ? b_id - (uint32_t)lo : 0xffffffffu;
    claim(d);
    for (int i = HB * NT + tid; r.hist && i < nh; i += NT) {
      uint32_t one[1] = {place(i, __ldg(ids + i))};
      claim(one);
    }
    for (int i = NT + tid; r.bias_id && i < r.n_bias; i += NT) {
      uint32_t one[1] = {__ldg(r.bias_id + row * r.bias_stride + i) - (uint32_t)lo};
      claim(one);
    }
    __syncthreads();
  }
#pragma unroll
  for (int k = 0; k < RUNS; k++) {
    const int i = (k * NT + tid) * V;
    if (i >= m) break;
    if (touch) {
#pragma unroll
      for (int q = 0; q < V; q += 4) {
        const int4 c = *reinterpret_cast<const int4 *>(cnt + i + q);
        const float4 f = *reinterpret_cast<const float4 *>(val + i + q);
        if (c.x < 0) v[k][q] = from_f<E>(f.x);
        if (c.y < 0) v[k][q + 1] = from_f<E>(f.y);
        if (c.z < 0) v[k][q + 2] = from_f<E>(f.z);
        if (c.w < 0) v[k][q + 3] = from_f<E>(f.w);
      }
    }
    if (allow) {
#pragma unroll
      for (int e = 0; e < V; e++)
        if (!((ok[k] >> e) & 1)) v[k][e] = from_f<E>(-CUDART_INF_F);
    }
    if (vec && i + V <= m) {
      *reinterpret_cast<uint4 *>(y + i) = *reinterpret_cast<const uint4 *>(v[k]);
    } else {
#pragma unroll
      for (int e = 0; e < V; e++)
        if (i + e < m) y[i + e] = v[k][e];
    }
  }
}

// 16 bytes that are read once: no room in L1.
template <class E>
__device__ __forceinline__ uint4 ld_stream(const E *p) {
  uint4 v;
  asm volatile("ld.global.L1::no_allocate.v4.u32 {%0,%1,%2,%3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "l"(p) : "memory");
  return v;
}

// The usual case, lists of up to a few thousand ids: a CTA takes a part of a
// row.  Half of its warps put the tokens of the part that the lists name into
// a hash table in shared memory (counts, biases) and finish them from there,
// while the others already stream the part through with nothing but the mask;
// then all stream what is left, and the finished ones go to their places.
// What streams is the logit itself or, where it is masked, -inf, so in place
// too a logit that a rule still reads is either untouched or not needed.
// Every part reads the whole lists, so a row has as many parts as fill the
// SMs and no more.  250 rows of 128256 with 3000 ids and 300 biases: 95 us
// with counts for every token of a segment of 8192, 80 us with the table
// before the stream, 64 us beside it (the copy alone: 42 us).
template <int T, int NT, int CTAS>
__global__ void __launch_bounds__(NT, CTAS) k_logit_rules_hash(const void *in, void *out, int n, long in_stride, long out_stride,
                                                               const pk_logit_rules r, int parts, int part_len, int bits, int vec) {
  using E = elem_t<T>;
  constexpr int V = 16 / (int)sizeof(E), RUNS = 4, CHUNK = RUNS * 32 * V;  // a warp's runs in flight
  constexpr int NB = NT / 2;  // threads that build
  extern __shared__ __align__(16) uint8_t smem[];
  const int slots = r.hist || r.bias_id ? 1 << bits : 0;
  uint32_t *tab = reinterpret_cast<uint32_t *>(smem);      // 0, or (place in the part + 1) << 16 | count
  float *val = reinterpret_cast<float *>(smem) + slots;      // biases, then finished values
  __shared__ uint32_t bid[NB];
  __shared__ float bval[NB];
  __shared__ int bcount[NB / 32], next;
  pdl_trigger();
  pdl_wait();
  const int row = blockIdx.x / parts;
  const int lo = (int)(blockIdx.x - row * parts) * part_len, m = min(part_len, n - lo), tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const E *x = reinterpret_cast<const E *>(in) + row * in_stride + lo;
  E *y = reinterpret_cast<E *>(out) + row * out_stride + lo;
  const uint32_t *allow = r.allow ? r.allow + row * r.allow_stride + (lo >> 5) : nullptr;  // (parts start at whole words)
  if (tid == 0) next = 0;
  for (int i = tid; i < 2 * slots / 4; i += NT) reinterpret_cast<uint4 *>(smem)[i] = make_uint4(0, 0, 0, 0);
  __syncthreads();
  if (slots && tid < NB) {
    auto sync = [] { asm volatile("bar.sync 1, %0;" ::"n"(NB) : "memory"); };  // of the building threads
    // adds `times` to place d's count; its slot.  The table has room for every
    // entry of the lists, so a free slot is met before all were tried.
    auto enter = [&](uint32_t d, uint32_t times) {
      const uint32_t mine = (d + 1) << 16;
      uint32_t h = (d * 0x9e3779b1u) >> (32 - bits);
      for (int probes = 0; probes < slots; probes++) {
        uint32_t k = *(volatile uint32_t *)(tab + h);
        if (k == 0) {
          k = atomicCAS(tab + h, 0u, mine + times);
          if (k == 0) break;
        }
        if ((k & 0xffff0000u) == mine) {
          if (times) atomicAdd(tab + h, times);
          break;
        }
        h = (h + 1) & (slots - 1);
      }
      return h;
    };
    if (r.hist) {
      const int nh = min(max(r.n_hist ? __ldg(r.n_hist + row) : r.n_hist_max, 0), r.n_hist_max);
      constexpr int N = 8;  // ids at once: each wait is microseconds while the others stream
      for (int i0 = tid; i0 < nh; i0 += N * NB) {
        uint32_t d[N];
#pragma unroll
        for (int i = 0; i < N; i++) d[i] = i0 + i * NB < nh ? __ldg(r.hist + row * r.hist_stride + i0 + i * NB) - (uint32_t)lo : 0xffffffffu;
#pragma unroll 1
        for (int i = 0; i < N; i++) {
          uint32_t e = d[0];
#pragma unroll
          for (int j = 0; j + 1 < N; j++) d[j] = d[j + 1];
          if (e < (uint32_t)m) enter(e, 1);
        }
      }
    }
    for (int i0 = 0; r.bias_id && i0 < r.n_bias; i0 += NB) {  // (uniform)
      const int i = i0 + tid;
      const uint32_t d = i < r.n_bias ? __ldg(r.bias_id + row * r.bias_stride + i) - (uint32_t)lo : 0xffffffffu;
      const float b = i < r.n_bias ? __ldg(r.bias + row * r.bias_stride + i) : 0.0f;
      const bool mine = i < r.n_bias && d < (uint32_t)m;
      const unsigned here = __ballot_sync(0xffffffffu, mine);
      if (lane == 0) bcount[warp] = __popc(here);
      sync();
      int at = __popc(here & ((1u << lane) - 1)), all = 0;
#pragma unroll
      for (int w = 0; w < NB / 32; w++) {
        at += w < warp ? bcount[w] : 0;
        all += bcount[w];
      }
      if (mine) {
        bid[at] = enter(d, 0);
        bval[at] = b;
      }
      sync();
      if (warp == 0) {
        for (int j0 = 0; j0 < all; j0 += 32) {
          const uint32_t h = j0 + lane < all ? bid[j0 + lane] : 0xffffffffu;
          const unsigned same = __match_any_sync(0xffffffffu, h);
          if (h != 0xffffffffu) {
            for (unsigned left = same; left; left &= left - 1) {  // lanes with the same id, in order
              if (lane == __ffs(left) - 1) val[h] += bval[j0 + lane];
              __syncwarp(same);
            }
          }
          __syncwarp();
        }
      }
      sync();
    }
    const float rep = r.repeat ? __ldg(r.repeat + row) : 1.0f, fr = r.freq ? __ldg(r.freq + row) : 0.0f,
                pr = r.presence ? __ldg(r.presence + row) : 0.0f;
    sync();
    for (int h0 = tid; h0 < slots; h0 += 8 * NB) {  // eight slots' logits at once
      int d[8];
      float f[8];
      uint32_t w[8], c[8];
#pragma unroll
      for (int i = 0; i < 8; i++) {
        c[i] = h0 + i * NB < slots ? tab[h0 + i * NB] : 0;
        d[i] = (int)(c[i] >> 16) - 1;
        f[i] = d[i] >= 0 ? to_f(*(const volatile E *)(x + d[i])) : 0.0f;
        w[i] = d[i] >= 0 && allow ? __ldg(allow + (d[i] >> 5)) : 0xffffffffu;
      }
#pragma unroll
      for (int i = 0; i < 8; i++) {
        if (d[i] < 0) continue;
        const int h = h0 + i * NB, times = (int)(c[i] & 0xffffu);
        if (times > 0) {
          f[i] = f[i] > 0.0f ? fdiv(f[i], rep) : fmul(f[i], rep);
          f[i] = fsub(f[i], fadd(fmul((float)times, fr), pr));
        }
        val[h] = (w[i] >> (d[i] & 31)) & 1 ? fadd(f[i], val[h]) : -CUDART_INF_F;
      }
    }
  }
  __syncwarp();
  for (;;) {  // chunks of the part, as warps come for them
    int i0 = 0;
    if (lane == 0) i0 = atomicAdd(&next, CHUNK);
    i0 = __shfl_sync(0xffffffffu, i0, 0);
    if (i0 >= m) break;
    alignas(16) E v[RUNS][V];
    uint32_t ok[RUNS];
#pragma unroll
    for (int k = 0; k < RUNS; k++) {
      const int i = i0 + (k * 32 + lane) * V;
      ok[k] = 0xffffffffu;
      if (i >= m) continue;
      if (vec && i + V <= m) {
        *reinterpret_cast<uint4 *>(v[k]) = ld_stream(x + i);
      } else {
#pragma unroll
        for (int e = 0; e < V; e++)
          if (i + e < m) v[k][e] = x[i + e];
      }
      if (allow) ok[k] = __ldg(allow + (i >> 5)) >> (i & 31);  // V divides 32
    }
#pragma unroll
    for (int k = 0; k < RUNS; k++) {
      const int i = i0 + (k * 32 + lane) * V;
      if (i >= m) break;
      if (allow) {
#pragma unroll
        for (int e = 0; e < V; e++)
          if (!((ok[k] >> e) & 1)) v[k][e] = from_f<E>(-CUDART_INF_F);
      }
      if (vec && i + V <= m) {
        *reinterpret_cast<uint4 *>(y + i) = *reinterpret_cast<const uint4 *>(v[k]);
      } else {
#pragma unroll
        for (int e = 0; e < V; e++)
          if (i + e < m) y[i + e] = v[k][e];
      }
    }
  }
  if (slots) {
    __syncthreads();
    for (int h = tid; h < slots; h += NT)
      if (tab[h]) y[(tab[h] >> 16) - 1] = from_f<E>(val[h]);
  }
}

// 4096 slots of 8 bytes, so that three CTAs leave the SM's L1 room for the
// loads in flight (with 12 bytes and four CTAs: 89 us against 71).
constexpr int HASH_MOST = 12;
template <int T>
cudaError_t rules_type(const void *in, void *out, int rows, int n, long is, long os, const pk_logit_rules &r, cudaStream_t st) {
  constexpr int es = (int)sizeof(elem_t<T>), V = 16 / es, NT = 512, SEG = 8192;
  // a place and its one fit 16 bits, after a part is rounded up to whole runs of its threads too
  constexpr int MOST = 65536 / (NT * V) * (NT * V) - NT * V;
  static_assert(MOST % (NT * V) == 0 && MOST < 65535, "places of a part");
  const int vec = (((uintptr_t)in | (uintptr_t)out | (rows > 1 ? (uintptr_t)(is | os) * es : 0)) & 15) == 0;
  const long long entries = (r.hist ? r.n_hist_max : 0) + (long long)(r.bias_id ? r.n_bias : 0);
  int bits = 5;
  while (bits <= HASH_MOST && (1 << bits) < entries + entries / 5 + 1) bits++;
  if (bits <= HASH_MOST) {
    // parts of a row: about 592 CTAs (more read the lists more often: 75 us with 1000), none
    // smaller than its threads' first runs
    long long parts = std::max<long long>(1, std::min<long long>(592 / rows + 1, (n + 4 * NT - 1) / (4 * NT)));
    parts = std::max<long long>(parts, (n + MOST - 1) / MOST);
    const int len = (int)(((n + parts - 1) / parts + NT * V - 1) / (NT * V) * (NT * V));
    parts = (n + len - 1) / len;
    if (rows * parts > 0x7fffffffLL) return cudaErrorInvalidValue;
    const int smem = entries || r.hist || r.bias_id ? 8 << bits : 0;
    return launch(k_logit_rules_hash<T, NT, 3>, dim3((unsigned)(rows * parts)), dim3(NT), smem, st, in, out, n, is, os, r, (int)parts, len,
                  bits, vec);
  }
  const int segs = (n + SEG - 1) / SEG;
  const long long blocks = (long long)rows * segs;
  if (blocks > 0x7fffffffLL) return cudaErrorInvalidValue;
  return launch(k_logit_rules<T, SEG, 512, 3>, dim3((unsigned)blocks), dim3(512), 2 * SEG * 4, st, in, out, n, is, os, r, segs, vec);
}

}  // namespace

cudaError_t launch_rope(const pk_rope_args &a, cudaStream_t st) {
  return a.type == T_F32 ? rope_type<T_F32>(a, st) : a.type == T_F16 ? rope_type<T_F16>(a, st) : rope_type<T_BF16>(a, st);
}

cudaError_t launch_logit_rules(const void *logits, void *out, int type, int rows, int n, long in_stride,
                               long out_stride, const pk_logit_rules &r, cudaStream_t st) {
  return type == T_F32   ? rules_type<T_F32>(logits, out, rows, n, in_stride, out_stride, r, st)
         : type == T_F16 ? rules_type<T_F16>(logits, out, rows, n, in_stride, out_stride, r, st)
                         : rules_type<T_BF16>(logits, out, rows, n, in_stride, out_stride, r, st);
}

}  // namespace pk
