// pk_rows.cu -- kernels that go over rows once: rotary positions and the
// rules on logits.  The engine's own RoPE (k_rope_kv, model.rs:408-461) reads
// f32 tables of every position; these are the op level's, for any position.
#include <math_constants.h>

#include <algorithm>

#include "pk_cache.cuh"
#include "pk_cache.h"

namespace pk {
namespace {

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

// ------------------------------------------------------------------- rotary
// A CTA takes one token and some of its heads: the angles once for them all
// (double: position times turns, less its whole turns, is exact to 2^-53 of
// the angle; the remainder's cosine and sine in f32), while the first values
// are on their way.  An item is V elements (16 bytes where everything is
// aligned for it): for interleaved pairs a run of a head's dimensions, for
// the half layout V pairs' two runs, or a run that is copied.  A thread keeps
// its place in the head and goes from head to head, so its cosines and sines
// stay in registers and its addresses are additions (with an item's place
// divided out anew, index arithmetic was half the kernel's instructions).
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
                (size_t)(a.n_rot / 2) * sizeof(float2), st, a, per);
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
// A CTA takes SEG logits of a row, NT threads.  All that it reads (logits,
// masks, the first HB NT history ids, the first NT biases, the row's numbers)
// is asked for at the start, while its counts are cleared, so that it waits
// for memory once; asked for where it is used, that was five times in a row
// and 97 us for 250 rows of 128256.  It counts the row's ids that fall into
// its segment in shared memory (whole counts: their order does not matter)
// and collects the biases of the segment there, in the list's order, which
// one warp adds up; then the segment is finished and written.
template <int T, int SEG, int NT>
__global__ void __launch_bounds__(NT) k_logit_rules(const void *in, void *out, int n, long in_stride, long out_stride,
                                                    const pk_logit_rules r, int segs, int vec) {
  using E = elem_t<T>;
  constexpr int V = 16 / (int)sizeof(E), RUNS = SEG / (NT * V);  // a thread has runs of V elements
  constexpr int HB = 6;
  static_assert(RUNS * NT * V == SEG, "whole runs");
  extern __shared__ __align__(16) uint8_t smem[];
  int *cnt = reinterpret_cast<int *>(smem);                             // [SEG], where there is a history
  float *bias = reinterpret_cast<float *>(smem) + (r.hist ? SEG : 0);   // [SEG], where there are biases
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
  alignas(16) E v[RUNS][V];
  uint32_t ok[RUNS], hid[HB];
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
      hid[h] = 0xffffffffu;
      if (h * NT + tid < r.n_hist_max) hid[h] = __ldg(ids + h * NT + tid);
    }
  }
  uint32_t b_id = 0xffffffffu;
  float b_val = 0.0f;
  if (r.bias_id && tid < r.n_bias) {
    b_id = __ldg(r.bias_id + row * r.bias_stride + tid);
    b_val = __ldg(r.bias + row * r.bias_stride + tid);
  }
  const float rep = r.repeat ? __ldg(r.repeat + row) : 1.0f, fr = r.freq ? __ldg(r.freq + row) : 0.0f,
              pr = r.presence ? __ldg(r.presence + row) : 0.0f;
  const int words = (r.hist ? SEG : 0) + (r.bias_id ? SEG : 0);
  for (int i = tid; i < words / 4; i += NT) reinterpret_cast<uint4 *>(smem)[i] = make_uint4(0, 0, 0, 0);
  __syncthreads();
  if (r.hist) {
    nh = min(max(nh, 0), r.n_hist_max);
#pragma unroll
    for (int h = 0; h < HB; h++) {
      const uint32_t d = hid[h] - (uint32_t)lo;
      if (h * NT + tid < nh && d < (uint32_t)m) atomicAdd(&cnt[d], 1);
    }
    for (int i = HB * NT + tid; i < nh; i += NT) {
      const uint32_t d = __ldg(ids + i) - (uint32_t)lo;
      if (d < (uint32_t)m) atomicAdd(&cnt[d], 1);
    }
  }
  if (r.bias_id) {
    for (int i0 = 0; i0 < r.n_bias; i0 += NT) {  // (uniform)
      if (i0 > 0) {
        const int i = i0 + tid;
        b_id = i < r.n_bias ? __ldg(r.bias_id + row * r.bias_stride + i) : 0xffffffffu;
        b_val = i < r.n_bias ? __ldg(r.bias + row * r.bias_stride + i) : 0.0f;
      }
      const uint32_t d = i0 + tid < r.n_bias ? b_id - (uint32_t)lo : 0xffffffffu;
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
        bval[at] = b_val;
      }
      __syncthreads();
      if (warp == 0) {
        for (int j0 = 0; j0 < all; j0 += 32) {
          const uint32_t id = j0 + lane < all ? bid[j0 + lane] : 0xffffffffu;
          const unsigned same = __match_any_sync(0xffffffffu, id);
          if (id != 0xffffffffu) {
            for (unsigned left = same; left; left &= left - 1) {  // lanes with the same id, in order
              if (lane == __ffs(left) - 1) bias[id] += bval[j0 + lane];
              __syncwarp(same);
            }
          }
          __syncwarp();
        }
      }
      __syncthreads();
    }
  }
  __syncthreads();
#pragma unroll
  for (int k = 0; k < RUNS; k++) {
    const int i = (k * NT + tid) * V;
    if (i >= m) break;
    // most runs have no token that was seen or biased
#pragma unroll
    for (int q = 0; q < V; q += 4) {
      int4 c = make_int4(0, 0, 0, 0);
      float4 b = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
      if (r.hist) c = *reinterpret_cast<const int4 *>(cnt + i + q);
      if (r.bias_id) b = *reinterpret_cast<const float4 *>(bias + i + q);
      const int cc[4] = {c.x, c.y, c.z, c.w};
      const float bb[4] = {b.x, b.y, b.z, b.w};
      if (c.x | c.y | c.z | c.w | __float_as_int(b.x) | __float_as_int(b.y) | __float_as_int(b.z) | __float_as_int(b.w)) {
#pragma unroll
        for (int e = 0; e < 4; e++) {
          float f = to_f(v[k][q + e]);
          if (cc[e] > 0) {
            f = f > 0.0f ? fdiv(f, rep) : fmul(f, rep);
            f = fsub(f, fadd(fmul((float)cc[e], fr), pr));
          }
          v[k][q + e] = from_f<E>(fadd(f, bb[e]));
        }
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

template <int T, int SEG, int NT>
cudaError_t rules_as(const void *in, void *out, int rows, int n, long is, long os, const pk_logit_rules &r, cudaStream_t st) {
  constexpr int es = (int)sizeof(elem_t<T>);
  const int segs = (n + SEG - 1) / SEG;
  const long long blocks = (long long)rows * segs;
  if (blocks > 0x7fffffffLL) return cudaErrorInvalidValue;
  const int vec = (((uintptr_t)in | (uintptr_t)out | (rows > 1 ? (uintptr_t)(is | os) * es : 0)) & 15) == 0;
  const int smem = ((r.hist ? SEG : 0) + (r.bias_id ? SEG : 0)) * 4;
  const cudaError_t e = cudaFuncSetAttribute(k_logit_rules<T, SEG, NT>, cudaFuncAttributeMaxDynamicSharedMemorySize, 2 * SEG * 4);
  if (e != cudaSuccess) return e;
  return launch(k_logit_rules<T, SEG, NT>, dim3((unsigned)blocks), dim3(NT), (size_t)smem, st, in, out, n, is, os, r, segs, vec);
}
// Every CTA goes over the whole history, so segments are large (8192: 64 KB of
// counts and biases, three CTAs an SM) unless that leaves SMs idle.
template <int T>
cudaError_t rules_type(const void *in, void *out, int rows, int n, long is, long os, const pk_logit_rules &r, cudaStream_t st) {
  if ((long long)rows * ((n + 8191) / 8192) < 296) return rules_as<T, 2048, 256>(in, out, rows, n, is, os, r, st);
  return rules_as<T, 8192, 512>(in, out, rows, n, is, os, r, st);
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
