// pk_cache_attn.cu -- attention of new tokens (one, a causal run, or a drafted
// tree) over the quantised paged cache.  No counterpart in the reference,
// whose attention takes one token over an f32 cache (model.rs:993-1087).
//
// For a row (token i, query head h) over the positions t that it sees:
//   s_t = r D^K_t sum_d q'_d c^K_td      q = 2^e q', |q'| < 2, r = scale log2(e) 2^e
//   w_t = 2^(s_t - M)
//   out = sum_t w_t D^V_t c^V_t / sum_t w_t
// with integer codes c (|c| <= 128, exact in f16) and one f32 scale D a cache
// row, so the codes go to the matrix instructions (m16n8k16, f16 in, f32 sums)
// undequantised and the scales are applied outside them: D^K to the sums,
// D^V to the weights.  The products w D^V are rounded to f16, as fractions of
// the row's largest so far (a large V row with a small weight must not push
// the others below f16's range); f32 queries are split into two f16 terms (22
// bits), and so are their products, those with the codes being exact.  M, the
// sums of w and the outputs are f32; M follows the running maximum only when
// that has grown by 2^6, so most tiles leave the outputs as they are.
//
// The contraction's order is free, so fragments are loaded straight from the
// cache rows: of 4 lanes that share a key each takes a quarter of its row's
// bytes as its k values, and of 8 lanes that share a position pair each takes
// an eighth of the V rows as its output dimensions.
#include <math_constants.h>

#include <algorithm>

#include "pk_cache.cuh"
#include "pk_cache.h"

namespace pk {
namespace {

constexpr float kLog2e = 1.4426950408889634f;
constexpr int MIN_CHUNK = 256;
// M moves when the maximum passes it by 2^GROW; a row's factor inv is set so
// that its largest weight times scale is SET and set again past TOP (f16 ends
// at 65504), so what rounds to a subnormal is below 2^-23 of the largest.
constexpr float GROW = 6.0f, SET = 512.0f, TOP = 32768.0f;

__device__ __forceinline__ void mma16816(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ uint32_t h2u(__half2 h) { return *reinterpret_cast<uint32_t *>(&h); }
__device__ __forceinline__ __half2 u2h(uint32_t u) { return *reinterpret_cast<__half2 *>(&u); }
// (a, b) as two f16 and, for the second term, what the rounding left.
__device__ __forceinline__ uint32_t pack2(float a, float b) { return h2u(__floats2half2_rn(a, b)); }
__device__ __forceinline__ uint32_t rest2(float a, float b, uint32_t hi) {
  const float2 f = __half22float2(u2h(hi));
  return pack2(a - f.x, b - f.y);
}

// Over the four lanes that share a row.
__device__ __forceinline__ float quad_max(float v) {
  v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, 1));
  return fmaxf(v, __shfl_xor_sync(0xffffffffu, v, 2));
}

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

struct AttnKArgs {
  pk_kv_cache c;
  pk_kv_seqs s;
  pk_kv_query q;
  float *part_o;   // [n_tok][n_head][n_chunk][DH]
  float2 *part_ml; // [n_tok][n_head][n_chunk]
  int chunk, n_chunk, row_tiles, group, vec_q, vec_o;
};

// Positions of a row tile's chunk, and whether the sequence's rows come from
// more than one chunk (then this one's go to the scratch).
struct Unit {
  SeqView sv;
  int s, h, rt, ch, lo, hi, nch, rows;
};

// DH / 4 query elements of a row from lane t's quarter, scaled to |q'| < 2;
// rs is the row's r.  All lanes of the warp call it.
template <int DH, class E>
__device__ __forceinline__ void load_q(const AttnKArgs &a, const Unit &u, int row, int t, float (&x)[DH / 4], float &rs) {
  const bool on = row < u.rows;
  const int i = row / a.group, h = u.h * a.group + row - i * a.group;
  if (on) {
    const E *p = reinterpret_cast<const E *>(a.q.q) + (long long)(u.sv.first + i) * a.q.q_tok_stride +
                 (long long)h * a.q.q_head_stride + t * (DH / 4);
    load_n<E, DH / 4>(p, a.vec_q, x);
  }
  float m = 0.0f;
#pragma unroll
  for (int j = 0; j < DH / 4; j++) {
    if (!on) x[j] = 0.0f;
    m = fmaxf(m, fabsf(x[j]));
  }
  m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, 1));
  m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, 2));
  int e = (int)(__float_as_uint(m) >> 23) - 127;  // m in [2^e, 2^(e+1))
  e = m > 0.0f ? min(max(e, -100), 126) : 0;
  const float up = __int_as_float((e + 127) << 23), down = __int_as_float((127 - e) << 23);
#pragma unroll
  for (int j = 0; j < DH / 4; j++) x[j] *= down;
  rs = a.q.scale * kLog2e * up;
}

template <int DH>
__device__ __forceinline__ void load_q_any(const AttnKArgs &a, const Unit &u, int row, int t, float (&x)[DH / 4], float &rs) {
  if (a.q.type == T_F32) load_q<DH, float>(a, u, row, t, x, rs);
  else if (a.q.type == T_F16) load_q<DH, __half>(a, u, row, t, x, rs);
  else load_q<DH, __nv_bfloat16>(a, u, row, t, x, rs);
}

// The k slots' dimensions within a lane's quarter: k step j's four values are
// elements dim_of(j, 0..3).  Q8: four bytes of a word; Q4: nibble pairs
// (i, i + 4) of a word of eight.
template <int TYPE>
__host__ __device__ constexpr int dim_of(int j, int e) {
  return TYPE == PK_KV_Q8 ? 4 * j + e : 8 * (j / 2) + 2 * (j % 2) + (e / 2) + 4 * (e % 2);
}

// Does row (token i) see draft j?
__device__ __forceinline__ bool sees(const AttnKArgs &a, const Unit &u, int i, int j) {
  if (j >= u.sv.n) return false;
  if (!a.q.mask) return j <= i;
  if ((j >> 6) >= a.q.mask_words) return false;
  return (__ldg(a.q.mask + (size_t)(u.sv.first + i) * a.q.mask_words + (j >> 6)) >> (j & 63)) & 1;
}

// One warp's state: 16 rows (lane's rows g and g + 8) over some positions.
template <int TYPE, int DH, int NT>
struct Warp {
  static constexpr int KS = DH / 16, NV = DH / 8;
  static constexpr int RB = TYPE == PK_KV_Q8 ? DH : DH / 2, SW = TYPE == PK_KV_Q8 ? 1 : 2;
  uint32_t q[NT][KS][4];
  float o[NV][4];
  float rs[2], m[2], l[2], inv[2];

  __device__ __forceinline__ void init(const AttnKArgs &a, const Unit &u, int row0, int lane) {
    const int g = lane >> 2, t = lane & 3;
#pragma unroll
    for (int r = 0; r < 2; r++) {
      float x[DH / 4];
      load_q_any<DH>(a, u, row0 + g + 8 * r, t, x, rs[r]);
#pragma unroll
      for (int j = 0; j < KS; j++) {
#pragma unroll
        for (int e = 0; e < 2; e++) {
          const float x0 = x[dim_of<TYPE>(j, 2 * e)], x1 = x[dim_of<TYPE>(j, 2 * e + 1)];
          q[0][j][r + 2 * e] = pack2(x0, x1);
          if (NT == 2) q[NT - 1][j][r + 2 * e] = rest2(x0, x1, q[0][j][r + 2 * e]);
        }
      }
      m[r] = -CUDART_INF_F;
      l[r] = 0.0f;
      inv[r] = 0x1p100f;
    }
#pragma unroll
    for (int i = 0; i < NV; i++) o[i][0] = o[i][1] = o[i][2] = o[i][3] = 0.0f;
  }

  __device__ __forceinline__ void scale_row(int r, float f) {
#pragma unroll
    for (int i = 0; i < NV; i++) {
      o[i][2 * r] *= f;
      o[i][2 * r + 1] *= f;
    }
  }

  // Sixteen positions p0 .. p0 + 15 (one page's rows from `row`, or row < 0).
  // masked: some of them may be out of reach of some row.
  __device__ __forceinline__ void tile(const AttnKArgs &a, const Unit &u, int row0, int p0, long long row, bool masked,
                                       int lane) {
    const int g = lane >> 2, t = lane & 3;
    const uint8_t *kc = reinterpret_cast<const uint8_t *>(a.c.k) + (size_t)row * RB;
    const uint8_t *vc = reinterpret_cast<const uint8_t *>(a.c.v) + (size_t)row * RB;
    const float *ks = a.c.ks + (size_t)row * SW, *vs = a.c.vs + (size_t)row * SW;
    float s[2][4];
#pragma unroll
    for (int n = 0; n < 2; n++) {
      s[n][0] = s[n][1] = s[n][2] = s[n][3] = 0.0f;
      const uint8_t *kp = kc + (size_t)(8 * n + g) * RB + t * (RB / 4);
      uint32_t w[RB / 16];
      if (RB / 4 >= 16) {
#pragma unroll
        for (int i = 0; i < RB / 64; i++) *reinterpret_cast<uint4 *>(w + 4 * i) = reinterpret_cast<const uint4 *>(kp)[i];
      } else {
        *reinterpret_cast<uint2 *>(w) = *reinterpret_cast<const uint2 *>(kp);
      }
      uint32_t sub = 0, sd = 0, md = 0;
      if (TYPE == PK_KV_Q4) {
        sub = __float_as_uint(ks[2 * (8 * n + g) + 1]);
        const int sb = (int)((sub >> (4 * (t * (DH / 4) / 32))) & 15u);
        sd = dup_h(sb);
        md = dup_h(-1032 * sb);
      }
#pragma unroll
      for (int j = 0; j < KS; j++) {
        uint32_t b0, b1;
        if (TYPE == PK_KV_Q8) {
          b0 = codes_of(w[j], 0x4140);
          b1 = codes_of(w[j], 0x4342);
        } else {
          b0 = nibbles_of(w[j / 2] >> (8 * (j % 2)), sd, md);
          b1 = nibbles_of(w[j / 2] >> (8 * (j % 2) + 4), sd, md);
        }
        mma16816(s[n], q[0][j], b0, b1);
        if (NT == 2) mma16816(s[n], q[NT - 1][j], b0, b1);
      }
    }
    // this lane's columns: positions p0 + 8 n + 2 t + {0, 1}
    float dk[2][2], dv[2][2];
    uint32_t vsub[2][2];
#pragma unroll
    for (int n = 0; n < 2; n++) {
#pragma unroll
      for (int e = 0; e < 2; e++) {
        const int k = 8 * n + 2 * t + e;
        dk[n][e] = ks[k * SW];
        dv[n][e] = vs[k * SW];
        if (TYPE == PK_KV_Q4) vsub[n][e] = __float_as_uint(vs[k * SW + SW - 1]);
      }
    }
    bool vis[2][2][2];  // by n-tile, column, row
    if (masked) {
#pragma unroll
      for (int n = 0; n < 2; n++)
#pragma unroll
        for (int e = 0; e < 2; e++) {
          const int p = p0 + 8 * n + 2 * t + e;
#pragma unroll
          for (int r = 0; r < 2; r++) {
            const int rr = row0 + g + 8 * r;
            vis[n][e][r] = p < u.hi && rr < u.rows && (p < u.sv.ctx || sees(a, u, rr / a.group, p - u.sv.ctx));
          }
        }
    }
    float mx[2];
#pragma unroll
    for (int r = 0; r < 2; r++) {
#pragma unroll
      for (int n = 0; n < 2; n++)
#pragma unroll
        for (int e = 0; e < 2; e++) {
          const float v = s[n][2 * r + e] * dk[n][e] * rs[r];
          s[n][2 * r + e] = masked && !vis[n][e][r] ? -CUDART_INF_F : v;
        }
      mx[r] = quad_max(fmaxf(fmaxf(s[0][2 * r], s[0][2 * r + 1]), fmaxf(s[1][2 * r], s[1][2 * r + 1])));
    }
    // m starts at -inf: a row's first position is always more
    const bool grow0 = mx[0] > m[0] + GROW, grow1 = mx[1] > m[1] + GROW;
    if (__any_sync(0xffffffffu, grow0 || grow1)) {
#pragma unroll
      for (int r = 0; r < 2; r++) {
        if (!(r ? grow1 : grow0)) continue;
        l[r] *= ex2(m[r] - mx[r]);
        // what o holds shrinks by the same factor, which goes into inv; past
        // 2^100 (at the first position, from infinity) into o
        const float f = inv[r] * ex2(mx[r] - m[r]);
        m[r] = mx[r];
        inv[r] = fminf(f, 0x1p100f);
        if (f > 0x1p100f) scale_row(r, 0x1p100f / f);
      }
    }
    float xm[2];
#pragma unroll
    for (int r = 0; r < 2; r++) {
      const float mu = m[r] == -CUDART_INF_F ? 0.0f : m[r];
      xm[r] = 0.0f;
#pragma unroll
      for (int n = 0; n < 2; n++)
#pragma unroll
        for (int e = 0; e < 2; e++) {
          const float p = ex2(s[n][2 * r + e] - mu);
          l[r] += p;
          const float x = masked && !vis[n][e][r] ? 0.0f : p * dv[n][e];
          s[n][2 * r + e] = x;
          xm[r] = fmaxf(xm[r], x);
        }
      xm[r] = quad_max(xm[r]);
    }
    const bool big0 = xm[0] * inv[0] > TOP, big1 = xm[1] * inv[1] > TOP;
    if (__any_sync(0xffffffffu, big0 || big1)) {
#pragma unroll
      for (int r = 0; r < 2; r++) {
        if (!(r ? big1 : big0)) continue;
        const float now = SET / fmaxf(xm[r], 0x1p-100f);
        scale_row(r, now / inv[r]);
        inv[r] = now;
      }
    }
    uint32_t ph[NT][4];
#pragma unroll
    for (int r = 0; r < 2; r++) {
#pragma unroll
      for (int n = 0; n < 2; n++) {
        const float x0 = s[n][2 * r] * inv[r], x1 = s[n][2 * r + 1] * inv[r];
        ph[0][r + 2 * n] = pack2(x0, x1);
        if (NT == 2) ph[NT - 1][r + 2 * n] = rest2(x0, x1, ph[0][r + 2 * n]);
      }
    }
    // V: this lane's DH / 8 dimensions of the four positions of its columns
    constexpr int VB = RB / 8, VW = VB / 4;
    uint32_t v[2][2][VW];
#pragma unroll
    for (int n = 0; n < 2; n++)
#pragma unroll
      for (int e = 0; e < 2; e++) {
        const uint8_t *vp = vc + (size_t)(8 * n + 2 * t + e) * RB + g * VB;
        if (VB == 16) *reinterpret_cast<uint4 *>(v[n][e]) = *reinterpret_cast<const uint4 *>(vp);
        else if (VB == 8) *reinterpret_cast<uint2 *>(v[n][e]) = *reinterpret_cast<const uint2 *>(vp);
        else v[n][e][0] = *reinterpret_cast<const uint32_t *>(vp);
      }
    uint32_t sd[2] = {0, 0}, md[2] = {0, 0};
    if (TYPE == PK_KV_Q4) {
      const int sh = 4 * (g * (DH / 8) / 32);
#pragma unroll
      for (int n = 0; n < 2; n++) {
        const int s0 = (int)((vsub[n][0] >> sh) & 15u), s1 = (int)((vsub[n][1] >> sh) & 15u);
        sd[n] = h2u(__halves2half2(__int2half_rn(s0), __int2half_rn(s1)));
        md[n] = h2u(__halves2half2(__int2half_rn(-1032 * s0), __int2half_rn(-1032 * s1)));
      }
    }
#pragma unroll
    for (int w = 0; w < VW; w++) {
      if (TYPE == PK_KV_Q8) {
        uint32_t x[2][2];
#pragma unroll
        for (int n = 0; n < 2; n++) {
          x[n][0] = __byte_perm(v[n][0][w], v[n][1][w], 0x5140);
          x[n][1] = __byte_perm(v[n][0][w], v[n][1][w], 0x7362);
        }
#pragma unroll
        for (int d = 0; d < 4; d++) {
          const uint32_t sel = d & 1 ? 0x4342 : 0x4140;
          const uint32_t b0 = codes_of(x[0][d / 2], sel), b1 = codes_of(x[1][d / 2], sel);
          mma16816(o[4 * w + d], ph[0], b0, b1);
          if (NT == 2) mma16816(o[4 * w + d], ph[NT - 1], b0, b1);
        }
      } else {
        uint32_t x[2][2];
#pragma unroll
        for (int n = 0; n < 2; n++) {
          x[n][0] = __byte_perm(v[n][0][w], v[n][1][w], 0x5410);
          x[n][1] = __byte_perm(v[n][0][w], v[n][1][w], 0x7632);
        }
#pragma unroll
        for (int d = 0; d < 8; d++) {
          const uint32_t b0 = nibbles_of(x[0][d / 4] >> (4 * (d % 4)), sd[0], md[0]);
          const uint32_t b1 = nibbles_of(x[1][d / 4] >> (4 * (d % 4)), sd[1], md[1]);
          mma16816(o[8 * w + d], ph[0], b0, b1);
          if (NT == 2) mma16816(o[8 * w + d], ph[NT - 1], b0, b1);
        }
      }
    }
  }
};

__device__ __forceinline__ Unit unit_of(const AttnKArgs &a, int rows_tile) {
  Unit u;
  long long id = blockIdx.x;
  u.rt = (int)(id % a.row_tiles);
  id /= a.row_tiles;
  u.h = (int)(id % a.c.n_kv);
  id /= a.c.n_kv;
  u.ch = (int)(id % a.n_chunk);
  u.s = (int)(id / a.n_chunk);
  u.sv = seq_view(a.s, a.c.page_size, u.s);
  u.rows = u.sv.n * a.group;
  u.nch = (u.sv.total + a.chunk - 1) / a.chunk;
  u.lo = u.ch * a.chunk;
  u.hi = min(u.sv.total, u.lo + a.chunk);
  return u;
}

// Writes element pairs of lane's rows: the final row, or the chunk's part.
template <int DH>
__device__ __forceinline__ void write_row(const AttnKArgs &a, const Unit &u, int row, int d0, const float *x) {
  const int i = row / a.group, h = u.h * a.group + row - i * a.group;
  const long long tok = u.sv.first + i;
  if (u.nch > 1) {
    float *p = a.part_o + ((tok * a.q.n_head + h) * a.n_chunk + u.ch) * DH + d0;
#pragma unroll
    for (int j = 0; j < DH / 8; j += 4) *reinterpret_cast<float4 *>(p + j) = make_float4(x[j], x[j + 1], x[j + 2], x[j + 3]);
    return;
  }
  const long long off = tok * a.q.out_tok_stride + (long long)h * a.q.out_head_stride + d0;
  float v[DH / 8];
#pragma unroll
  for (int j = 0; j < DH / 8; j++) v[j] = x[j];
  if (a.q.type == T_F32) store_n<float, DH / 8>(reinterpret_cast<float *>(a.q.out) + off, a.vec_o, v);
  else if (a.q.type == T_F16) store_n<__half, DH / 8>(reinterpret_cast<__half *>(a.q.out) + off, a.vec_o, v);
  else store_n<__nv_bfloat16, DH / 8>(reinterpret_cast<__nv_bfloat16 *>(a.q.out) + off, a.vec_o, v);
}

// A CTA: 16 rows of one kv head of one sequence over one chunk of positions;
// its warps take tiles of 16 positions in turn and add up at the end.
constexpr int AW = 4;
template <int TYPE, int DH, int NT>
__global__ void __launch_bounds__(32 * AW) k_kv_attn(const AttnKArgs a) {
  __shared__ float so[AW][16][DH];
  __shared__ float sm[AW][16], sl[AW][16];
  pdl_trigger();
  pdl_wait();
  const Unit u = unit_of(a, 16);
  const int row0 = u.rt * 16;
  if (u.ch >= max(u.nch, 1) || row0 >= u.rows) return;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, g = lane >> 2, t = lane & 3;
  Warp<TYPE, DH, NT> W;
  W.init(a, u, row0, lane);
  for (int p0 = u.lo + 16 * warp; p0 < u.hi; p0 += 16 * AW) {
    const long long row = row_at(a.c, a.s, u.s, p0, u.h);
    if (row < 0) continue;
    W.tile(a, u, row0, p0, row, p0 + 16 > min(u.sv.ctx, u.hi), lane);
  }
#pragma unroll
  for (int r = 0; r < 2; r++) {
    W.l[r] += __shfl_xor_sync(0xffffffffu, W.l[r], 1);
    W.l[r] += __shfl_xor_sync(0xffffffffu, W.l[r], 2);
    if (t == 0) {
      sm[warp][g + 8 * r] = W.m[r];
      sl[warp][g + 8 * r] = W.l[r];
    }
#pragma unroll
    for (int e = 0; e < 2; e++)
#pragma unroll
      for (int i = 0; i < DH / 8; i++) so[warp][g + 8 * r][(2 * t + e) * (DH / 8) + i] = W.o[i][2 * r + e] / W.inv[r];
  }
  __syncthreads();
  for (int x = threadIdx.x; x < 16 * 8; x += 32 * AW) {
    const int r = x >> 3, d0 = (x & 7) * (DH / 8);
    if (row0 + r >= u.rows) continue;
    float M = -CUDART_INF_F, L = 0.0f, acc[DH / 8];
#pragma unroll
    for (int w = 0; w < AW; w++) M = fmaxf(M, sm[w][r]);
#pragma unroll
    for (int j = 0; j < DH / 8; j++) acc[j] = 0.0f;
#pragma unroll
    for (int w = 0; w < AW; w++) {
      const float f = sl[w][r] == 0.0f ? 0.0f : ex2(sm[w][r] - M);  // a NaN sum stays one
      L = fmaf(f, sl[w][r], L);
#pragma unroll
      for (int j = 0; j < DH / 8; j++) acc[j] = fmaf(f, so[w][r][d0 + j], acc[j]);
    }
    if (u.nch > 1) {
      if ((x & 7) == 0) {
        const int i = (row0 + r) / a.group, h = u.h * a.group + (row0 + r) - i * a.group;
        a.part_ml[((long long)(u.sv.first + i) * a.q.n_head + h) * a.n_chunk + u.ch] = make_float2(M, L);
      }
    } else {
      const float inv = L > 0.0f || isnan(L) ? 1.0f / L : 0.0f;
#pragma unroll
      for (int j = 0; j < DH / 8; j++) acc[j] *= inv;
    }
    write_row<DH>(a, u, row0 + r, d0, acc);
  }
}

// Adds up the chunks of rows that have more than one: a warp a row.
template <int DH>
__global__ void __launch_bounds__(128) k_kv_attn_join(const AttnKArgs a) {
  pdl_trigger();
  pdl_wait();
  const int lane = threadIdx.x & 31;
  const long long w = (long long)blockIdx.x * 4 + (threadIdx.x >> 5);
  const long long tok = w / a.q.n_head;
  const int h = (int)(w - tok * a.q.n_head);
  if (tok >= a.s.n_tok) return;
  const int s = seq_of(a.s, (int)tok, lane);
  if (s < 0) return;
  const SeqView sv = seq_view(a.s, a.c.page_size, s);
  const int nch = (sv.total + a.chunk - 1) / a.chunk;
  if (tok - sv.first >= sv.n || nch <= 1) return;
  const float2 *ml = a.part_ml + w * a.n_chunk;
  const float *po = a.part_o + w * a.n_chunk * DH;
  float M = -CUDART_INF_F;
  for (int c = lane; c < nch; c += 32) M = fmaxf(M, ml[c].x);
#pragma unroll
  for (int i = 16; i > 0; i >>= 1) M = fmaxf(M, __shfl_xor_sync(0xffffffffu, M, i));
  constexpr int V = DH / 32;
  float L = 0.0f, acc[V];
#pragma unroll
  for (int j = 0; j < V; j++) acc[j] = 0.0f;
  for (int c = 0; c < nch; c++) {
    const float2 x = ml[c];
    const float f = x.y == 0.0f ? 0.0f : ex2(x.x - M);
    L = fmaf(f, x.y, L);
    if (f == 0.0f) continue;
#pragma unroll
    for (int j = 0; j < V; j++) acc[j] = fmaf(f, po[(size_t)c * DH + V * lane + j], acc[j]);
  }
  const float inv = L > 0.0f || isnan(L) ? 1.0f / L : 0.0f;
  const long long off = tok * a.q.out_tok_stride + (long long)h * a.q.out_head_stride + V * lane;
#pragma unroll
  for (int j = 0; j < V; j++) {
    const float v = acc[j] * inv;
    if (a.q.type == T_F32) reinterpret_cast<float *>(a.q.out)[off + j] = v;
    else if (a.q.type == T_F16) reinterpret_cast<__half *>(a.q.out)[off + j] = __float2half_rn(v);
    else reinterpret_cast<__nv_bfloat16 *>(a.q.out)[off + j] = __float2bfloat16_rn(v);
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
void (*attn_kernel(int type))(AttnKArgs) {
  return type == T_F32 ? k_kv_attn<TYPE, DH, 2> : k_kv_attn<TYPE, DH, 1>;
}

}  // namespace

KvSplit kv_attn_split(const pk_kv_cache &c, const pk_kv_seqs &s, int n_head, int type) {
  KvSplit p;
  const int group = n_head / c.n_kv;
  p.row_tiles = (int)(((long long)s.max_new * group + 15) / 16);
  const long long units = (long long)s.n_seq * c.n_kv * p.row_tiles, want = 148 * 8;
  const long long most = (s.max_len + MIN_CHUNK - 1) / MIN_CHUNK;
  long long n = std::max<long long>(1, std::min(most, units ? want / units : 1));
  p.chunk = (int)std::min<long long>(((s.max_len + n - 1) / n + 63) / 64 * 64, 1 << 30);
  p.n_chunk = (int)((s.max_len + (long long)p.chunk - 1) / p.chunk);
  return p;
}

size_t kv_attn_scratch_bytes(const pk_kv_cache &c, const pk_kv_seqs &s, int n_head, int type) {
  const KvSplit p = kv_attn_split(c, s, n_head, type);
  if (p.n_chunk <= 1) return 0;
  return (size_t)s.n_tok * n_head * p.n_chunk * (c.head_dim + 2) * sizeof(float);
}

cudaError_t launch_kv_attn(const pk_kv_cache &c, const pk_kv_seqs &s, const pk_kv_query &q, void *scratch,
                           cudaStream_t st) {
  const KvSplit p = kv_attn_split(c, s, q.n_head, q.type);
  AttnKArgs a{};
  a.c = c; a.s = s; a.q = q;
  a.chunk = p.chunk; a.n_chunk = p.n_chunk; a.row_tiles = p.row_tiles;
  a.group = q.n_head / c.n_kv;
  const uintptr_t es = q.type == T_F32 ? 4 : 2;
  a.vec_q = (((uintptr_t)q.q | (uintptr_t)q.q_tok_stride * es | (uintptr_t)q.q_head_stride * es) & 15) == 0;
  a.vec_o = (((uintptr_t)q.out | (uintptr_t)q.out_tok_stride * es | (uintptr_t)q.out_head_stride * es) & 15) == 0;
  const size_t rows = (size_t)s.n_tok * q.n_head;
  a.part_o = reinterpret_cast<float *>(scratch);
  a.part_ml = p.n_chunk > 1 ? reinterpret_cast<float2 *>(a.part_o + rows * p.n_chunk * c.head_dim) : nullptr;
  const long long blocks = (long long)s.n_seq * c.n_kv * p.row_tiles * p.n_chunk, jb = ((long long)rows + 3) / 4;
  if (blocks > 0x7fffffffLL || jb > 0x7fffffffLL) return cudaErrorInvalidValue;
  void (*k)(AttnKArgs) = c.type == PK_KV_Q8
                             ? (c.head_dim == 64 ? attn_kernel<PK_KV_Q8, 64>(q.type) : attn_kernel<PK_KV_Q8, 128>(q.type))
                             : (c.head_dim == 64 ? attn_kernel<PK_KV_Q4, 64>(q.type) : attn_kernel<PK_KV_Q4, 128>(q.type));
  cudaError_t e = launch(k, dim3((unsigned)blocks), dim3(32 * AW), 0, st, a);
  if (e != cudaSuccess || p.n_chunk <= 1) return e;
  return launch(c.head_dim == 64 ? k_kv_attn_join<64> : k_kv_attn_join<128>, dim3((unsigned)jb), dim3(128), 0, st, a);
}

}  // namespace pk
