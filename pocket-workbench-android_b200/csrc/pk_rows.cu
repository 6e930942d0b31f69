// pk_rows.cu -- kernels that go over rows once: rotary positions and the
// rules on logits.  The engine's own RoPE (k_rope_kv, model.rs:408-461) reads
// f32 tables of every position; these are the op level's, for any position.
#include <math_constants.h>

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
// A CTA takes one token: the angles once for all heads (double: position
// times turns, less its whole turns, is exact to 2^-53 of the angle; the
// remainder's cosine and sine in f32), then every head's elements.
constexpr int RT = 256;
template <int T>
__global__ void __launch_bounds__(RT) k_rope(const pk_rope_args a) {
  using E = elem_t<T>;
  extern __shared__ float2 cs[];  // [n_rot / 2]
  pdl_trigger();
  pdl_wait();
  const long long t = blockIdx.x;
  const int half = a.n_rot / 2;
  const double pos = (double)__ldg(a.pos + t);
  for (int i = threadIdx.x; i < half; i += RT) {
    double x = pos * __ldg(a.turns + i);
    x -= rint(x);
    float s, c;
    sincospif(2.0f * (float)x, &s, &c);
    cs[i] = make_float2(c * a.gain, s * a.gain);
  }
  __syncthreads();
  const int per = a.head_dim - half, nq = a.q ? a.n_head : 0, heads = nq + (a.k ? a.n_kv : 0);  // work items a head
  for (int x = threadIdx.x; x < heads * per; x += RT) {
    const int hh = x / per, i = x - hh * per;
    const bool k = hh >= nq;
    const int h = k ? hh - nq : hh;
    const E *in = reinterpret_cast<const E *>(k ? a.k : a.q) + t * (k ? a.k_tok_stride : a.q_tok_stride) +
                  h * (k ? a.k_head_stride : a.q_head_stride);
    E *out = reinterpret_cast<E *>(k ? a.k_out : a.q_out) + t * (k ? a.ko_tok_stride : a.qo_tok_stride) +
             h * (k ? a.ko_head_stride : a.qo_head_stride);
    if (i >= half) {
      out[i + half] = in[i + half];
      continue;
    }
    const int d0 = a.layout == PK_ROPE_HALF ? i : 2 * i, d1 = a.layout == PK_ROPE_HALF ? i + half : 2 * i + 1;
    const float u = to_f(in[d0]), v = to_f(in[d1]);
    const float2 c = cs[i];
    out[d0] = from_f<E>(u * c.x - v * c.y);
    out[d1] = from_f<E>(u * c.y + v * c.x);
  }
}

// -------------------------------------------------------------- logit rules
// A CTA takes SEG logits of a row.  It counts the row's history ids that fall
// into its segment in shared memory (whole counts: their order does not
// matter), adds up the biases there in the list's order, and then goes over
// the segment once.
constexpr int LT = 256, SEG = 2048;
template <int T>
__global__ void __launch_bounds__(LT) k_logit_rules(const void *in, void *out, int n, long in_stride, long out_stride,
                                                    const pk_logit_rules r, int segs) {
  using E = elem_t<T>;
  __shared__ int cnt[SEG];
  __shared__ float bias[SEG];
  pdl_trigger();
  pdl_wait();
  const long long row = blockIdx.x / segs;
  const int lo = (int)(blockIdx.x - row * segs) * SEG, m = min(SEG, n - lo);
  for (int i = threadIdx.x; i < SEG; i += LT) {
    cnt[i] = 0;
    bias[i] = 0.0f;
  }
  __syncthreads();
  if (r.hist) {
    const uint32_t *ids = r.hist + row * r.hist_stride;
    const int nh = min(max(r.n_hist ? __ldg(r.n_hist + row) : r.n_hist_max, 0), r.n_hist_max);
    for (int i = threadIdx.x; i < nh; i += LT) {
      const uint32_t d = __ldg(ids + i) - (uint32_t)lo;
      if (d < (uint32_t)m) atomicAdd(&cnt[d], 1);
    }
  }
  if (r.bias_id && threadIdx.x < 32) {  // one warp, so that equal ids add up in order
    for (int i0 = 0; i0 < r.n_bias; i0 += 32) {
      const int i = i0 + threadIdx.x;
      const uint32_t d = i < r.n_bias ? __ldg(r.bias_id + row * r.bias_stride + i) - (uint32_t)lo : 0xffffffffu;
      const float b = i < r.n_bias ? __ldg(r.bias + row * r.bias_stride + i) : 0.0f;
      const unsigned same = __match_any_sync(0xffffffffu, d < (uint32_t)m ? d : 0xffffffffu);
      if (d < (uint32_t)m) {
        for (unsigned left = same; left; left &= left - 1) {  // the group's lanes in order
          if ((int)threadIdx.x == __ffs(left) - 1) bias[d] += b;
          __syncwarp(same);
        }
      }
      __syncwarp();
    }
  }
  __syncthreads();
  const float rep = r.repeat ? __ldg(r.repeat + row) : 1.0f, fr = r.freq ? __ldg(r.freq + row) : 0.0f,
              pr = r.presence ? __ldg(r.presence + row) : 0.0f;
  const E *x = reinterpret_cast<const E *>(in) + row * in_stride + lo;
  E *y = reinterpret_cast<E *>(out) + row * out_stride + lo;
  for (int i = threadIdx.x; i < m; i += LT) {
    float v = to_f(x[i]);
    const int c = cnt[i];
    if (c > 0) {
      v = v > 0.0f ? fdiv(v, rep) : fmul(v, rep);
      v = fsub(v, fadd(fmul((float)c, fr), pr));
    }
    v = fadd(v, bias[i]);
    if (r.allow && !((__ldg(r.allow + row * r.allow_stride + ((lo + i) >> 5)) >> (i & 31)) & 1)) v = -CUDART_INF_F;
    y[i] = from_f<E>(v);
  }
}

}  // namespace

cudaError_t launch_rope(const pk_rope_args &a, cudaStream_t st) {
  void (*k)(pk_rope_args) = a.type == T_F32 ? k_rope<T_F32> : a.type == T_F16 ? k_rope<T_F16> : k_rope<T_BF16>;
  return launch(k, dim3((unsigned)a.n_tok), dim3(RT), (size_t)(a.n_rot / 2) * sizeof(float2), st, a);
}

cudaError_t launch_logit_rules(const void *logits, void *out, int type, int rows, int n, long in_stride,
                               long out_stride, const pk_logit_rules &r, cudaStream_t st) {
  const int segs = (n + SEG - 1) / SEG;
  const long long blocks = (long long)rows * segs;
  if (blocks > 0x7fffffffLL) return cudaErrorInvalidValue;
  void (*k)(const void *, void *, int, long, long, pk_logit_rules, int) =
      type == T_F32 ? k_logit_rules<T_F32> : type == T_F16 ? k_logit_rules<T_F16> : k_logit_rules<T_BF16>;
  return launch(k, dim3((unsigned)blocks), dim3(LT), 0, st, logits, out, n, in_stride, out_stride, r, segs);
}

}  // namespace pk
