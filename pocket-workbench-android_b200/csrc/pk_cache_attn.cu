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
// The products are formed transposed, S^T = K Q^T and O^T = V^T P^T, with keys
// and dimensions as the instruction's 16 rows and query rows as its 8 columns:
// a kv head's query rows (one for a plain token of an ungrouped head, 8 for a
// group of 8) then cost matrix work in steps of 8, not 16, and each code that
// was made f16 serves every column.  The weights, made with a key a lane row,
// become the second product's operand by 8 x 8 register transposes.  The
// contraction's order is free, so fragments are loaded as the cache's rows
// lie: of 4 lanes that share a key each takes a quarter of its row's bytes as
// its k values, and of 8 lanes that share two keys each takes an eighth of
// the V rows as its output dimensions.
//
// Measured: one token at 1500 positions, 64 heads over 8 of 128, Q8: 10 us a
// call; 8 sequences at 16256, 36 heads of 64, f32, Q8: 139 to 149 us by the box,
// 71 to 66% of a copy's rate; f32 of head_dim 128 with many rows, which have no
// tcgen05 kernel: 8 sequences of 8000 with trees of 64, 64 heads over 8, Q8:
// 1,136 us (f16 there: 199).  What bounds it: memory for few rows, the matrix
// instructions' 550 TFLOP/s and the codes' conversion for many, which is why
// those go to pk_cache_attn_tc.cu.
#include <math_constants.h>

#include <algorithm>

#include "pk_cache_attn.cuh"
#include "pk_launch.h"

namespace pk {
namespace {

constexpr int MIN_CHUNK = 256;
constexpr int NSTAGE = 4;  // tiles of 16 positions in a key group's ring
__device__ __forceinline__ void mma16816(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
// The transpose of an 8 x 8 f16 matrix held two columns a lane.
__device__ __forceinline__ uint32_t transpose8(uint32_t x) {
  uint32_t y;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
  return y;
}
// A barrier of n threads (whole warps).
__device__ __forceinline__ void bar_n(int id, int n) { asm volatile("bar.sync %0, %1;" ::"r"(id), "r"(n) : "memory"); }
// Over the eight lanes that share two query rows.
__device__ __forceinline__ float key_max(float v) {
  v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, 4));
  v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, 8));
  return fmaxf(v, __shfl_xor_sync(0xffffffffu, v, 16));
}

// DH / 4 query elements of a row from lane t's quarter, scaled to |q'| < 2;
// rs is the row's r.  All lanes of the warp call it; the four lanes of a quad
// hold one row.
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
    x[j] = on ? inf_nan(x[j]) : 0.0f;
    m = fmaxf(m, fabsf(x[j]));
  }
  m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, 1));
  m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, 2));
  int e = (int)(__float_as_uint(m) >> 23) - 127;  // m in [2^e, 2^(e+1))
  e = m > 0.0f ? min(max(e, -100), 126) : 0;
  const float up = __int_as_float((e + 127) << 23), down = __int_as_float((127 - e) << 23);
#pragma unroll
  for (int j = 0; j < DH / 4; j++) x[j] *= down;
  rs = fmaxf(a.q.scale * kLog2e * up, 0x1p-149f);  // (not 0, times which a masked -inf would be NaN)
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

// A tile in shared memory: 16 rows of K codes, 16 of V codes, their scales.
// Rows lie in lines of 128 bytes whose 16-byte slots are exchanged by line, so
// that both the K reads (8 rows x 4 quarters) and the V reads (every second
// row x 8 eighths) of a warp touch every bank once.
template <int TYPE, int DH>
struct Tile {
  static constexpr int RB = TYPE == PK_KV_Q8 ? DH : DH / 2, SW = TYPE == PK_KV_Q8 ? 1 : 2;
  static constexpr int CODES = 16 * RB, SCALES = 16 * SW * 4;
  static constexpr int BYTES = 2 * (CODES + SCALES);
  static constexpr int KS = DH / 16;
  __device__ static __forceinline__ uint32_t at(int row, int byte) {  // of a K or V block
    constexpr int RPL = 128 / RB, CPR = RB / 16;
    const int line = row / RPL, x = RB == 128 ? line & 7 : (line & 3) * 2;
    return line * 128 + ((((row % RPL) * CPR + (byte >> 4)) ^ x) << 4) + (byte & 15);
  }
  // Copies of a key group's n threads (thread i) into the tile at dst.
  __device__ static __forceinline__ void copy(const pk_kv_cache &c, long long row, uint32_t dst, int i, int n) {
    const uint8_t *k = reinterpret_cast<const uint8_t *>(c.k) + row * RB, *v = reinterpret_cast<const uint8_t *>(c.v) + row * RB;
    constexpr int CH = CODES / 16, SC = SCALES / 16;
#pragma unroll
    for (int j = 0; j < CH; j += 32) {
      const int x = j + i;
      if (x < CH) {
        const uint32_t o = at(x / (RB / 16), (x % (RB / 16)) * 16);
        cp16(dst + o, k + 16 * x);
        cp16(dst + CODES + o, v + 16 * x);
      }
      if (n > 32) break;  // (more than one warp: the loop below)
    }
    if (n > 32) {
      for (int x = i + n; x < CH; x += n) {
        const uint32_t o = at(x / (RB / 16), (x % (RB / 16)) * 16);
        cp16(dst + o, k + 16 * x);
        cp16(dst + CODES + o, v + 16 * x);
      }
    }
    if (i < 2 * SC) {
      const float *s = (i < SC ? c.ks : c.vs) + row * SW + (i % SC) * 4;
      cp16(dst + 2 * CODES + 16 * i, s);
    }
  }
};

// One warp's state: 8 NB query rows (this lane's are 8 b + 2 t + {0, 1}) over
// some of the positions.  QS: the query fragments stay in shared memory, where
// registers would not hold them beside the outputs.
// It goes TS tiles at a time: a step's maxima over the lanes, its tests and
// its loop are as much work as a tile's products where there are few rows.
template <int TYPE, int DH, int NT, int NB>
struct Warp {
  using T = Tile<TYPE, DH>;
  static constexpr int KS = DH / 16, MV = DH / 16, RB = T::RB, SW = T::SW;
  static constexpr bool QS = NT * NB * KS * 2 > 64;
  static constexpr int TS = NB <= 2 ? 2 : 1;  // (the scores of two would not fit the registers beside 32 rows' outputs)
  static constexpr int QBYTES = QS ? NT * NB * KS * 32 * 8 : 0;
  uint32_t q[QS ? 1 : NT][QS ? 1 : NB][QS ? 1 : KS][2];
  uint32_t qs;  // shared address of this lane's fragments
  float o[NB][MV][4];
  float rs[NB][2], m[NB][2], l[NB][2], inv[NB][2];

  // store_q: this warp writes the fragments to shared memory at qsmem (its key
  // group's warps of the same rows write the same values).
  __device__ __forceinline__ void init(const AttnKArgs &a, const Unit &u, int row0, int lane, uint32_t qsmem) {
    const int g = lane >> 2, t = lane & 3;
    qs = qsmem + lane * 8;
#pragma unroll
    for (int b = 0; b < NB; b++) {
      float x[DH / 4], r;
      load_q_any<DH>(a, u, row0 + 8 * b + g, t, x, r);  // lanes of quad g: row g
#pragma unroll
      for (int e = 0; e < 2; e++) {
        rs[b][e] = __shfl_sync(0xffffffffu, r, 4 * (2 * t + e));
        m[b][e] = -CUDART_INF_F;
        l[b][e] = 0.0f;
        inv[b][e] = 0x1p100f;
      }
#pragma unroll
      for (int j = 0; j < KS; j++) {
        uint32_t f[NT][2];
#pragma unroll
        for (int e = 0; e < 2; e++) {
          const float x0 = x[dim_of<TYPE>(j, 2 * e)], x1 = x[dim_of<TYPE>(j, 2 * e + 1)];
          f[0][e] = pack2(x0, x1);
          if (NT == 2) f[NT - 1][e] = rest2(x0, x1, f[0][e]);
        }
#pragma unroll
        for (int n = 0; n < NT; n++) {
          if (QS) {
            asm volatile("st.shared.v2.u32 [%0], {%1,%2};" ::"r"(qs + (uint32_t)(((n * NB + b) * KS + j) * 256)), "r"(f[n][0]), "r"(f[n][1]) : "memory");
          } else {
            q[n][b][j][0] = f[n][0];
            q[n][b][j][1] = f[n][1];
          }
        }
      }
#pragma unroll
      for (int i = 0; i < MV; i++) o[b][i][0] = o[b][i][1] = o[b][i][2] = o[b][i][3] = 0.0f;
    }
  }
  __device__ __forceinline__ uint2 frag(int n, int b, int j) const {
    if (QS) return sld_v2(qs + (uint32_t)(((n * NB + b) * KS + j) * 256));
    return make_uint2(q[QS ? 0 : n][QS ? 0 : b][QS ? 0 : j][0], q[QS ? 0 : n][QS ? 0 : b][QS ? 0 : j][1]);
  }

  __device__ __forceinline__ void scale_row(int b, int e, float f) {
#pragma unroll
    for (int i = 0; i < MV; i++) {
      o[b][i][e] *= f;
      o[b][i][2 + e] *= f;
    }
  }

  // Positions p0 .. p0 + 16 TS - 1, in shared memory from sm on.  MASKED: some
  // of them may be out of reach of some row; bit n of `held`: tile n has a page.
  template <bool MASKED>
  __device__ __forceinline__ void tile(const AttnKArgs &a, const Unit &u, int row0, int p0, uint32_t sm, uint32_t held, int lane) {
    const int g = lane >> 2, t = lane & 3;
    float s[NB][TS][4];  // [2 n + e]: key g + 8 n of the tile, row 8 b + 2 t + e
    float dv[TS][2];
#pragma unroll
    for (int y = 0; y < TS; y++) {
      const uint32_t sy = sm + y * T::BYTES, ksc = sy + 2 * T::CODES, vsc = ksc + T::SCALES;
      uint32_t w[2][RB / 16], sd[2] = {0, 0}, md[2] = {0, 0};
      float dk[2];
#pragma unroll
      for (int n = 0; n < 2; n++) {  // keys g and g + 8
        const int row = 8 * n + g;
        if (RB / 4 >= 16) {
#pragma unroll
          for (int i = 0; i < RB / 64; i++) {
            const uint4 v = sld_v4(sy + T::at(row, t * (RB / 4) + 16 * i));
            w[n][4 * i] = v.x; w[n][4 * i + 1] = v.y; w[n][4 * i + 2] = v.z; w[n][4 * i + 3] = v.w;
          }
        } else {
          const uint2 v = sld_v2(sy + T::at(row, t * (RB / 4)));
          w[n][0] = v.x; w[n][1] = v.y;
        }
        if (TYPE == PK_KV_Q4) {
          const uint2 v = sld_v2(ksc + row * 8);
          dk[n] = __uint_as_float(v.x);
          const int sb = (int)((v.y >> (4 * (t * (DH / 4) / 32))) & 15u);
          sd[n] = dup_h(sb);
          md[n] = dup_h(-1032 * sb);
        } else {
          dk[n] = sld_f(ksc + row * 4);
        }
        dv[y][n] = sld_f(vsc + row * 4 * SW);
      }
      float lo[NT == 2 ? NB : 1][4];
#pragma unroll
      for (int b = 0; b < NB; b++) {
#pragma unroll
        for (int i = 0; i < 4; i++) {
          s[b][y][i] = 0.0f;
          if (NT == 2) lo[NT == 2 ? b : 0][i] = 0.0f;
        }
      }
#pragma unroll
      for (int j = 0; j < KS; j++) {
        uint32_t f[4];
#pragma unroll
        for (int n = 0; n < 2; n++) {
          if (TYPE == PK_KV_Q8) {
            f[n] = codes_of(w[n][j], 0x4140);
            f[2 + n] = codes_of(w[n][j], 0x4342);
          } else {
            f[n] = nibbles_of(w[n][j / 2] >> (8 * (j % 2)), sd[n], md[n]);
            f[2 + n] = nibbles_of(w[n][j / 2] >> (8 * (j % 2) + 4), sd[n], md[n]);
          }
        }
#pragma unroll
        for (int b = 0; b < NB; b++) {
          const uint2 x = frag(0, b, j);
          mma16816(s[b][y], f, x.x, x.y);
          if (NT == 2) {  // small terms in sums of their own
            const uint2 v = frag(NT - 1, b, j);
            mma16816(lo[NT == 2 ? b : 0], f, v.x, v.y);
          }
        }
      }
#pragma unroll
      for (int b = 0; b < NB; b++)
#pragma unroll
        for (int i = 0; i < 4; i++) s[b][y][i] = (NT == 2 ? s[b][y][i] + lo[NT == 2 ? b : 0][i] : s[b][y][i]) * dk[i >> 1];
    }
    uint32_t seen[TS];  // bit 4 b + 2 n + e
    if (MASKED) {
#pragma unroll
      for (int y = 0; y < TS; y++) {
        seen[y] = 0;
#pragma unroll
        for (int b = 0; b < NB; b++)
#pragma unroll
          for (int e = 0; e < 2; e++) {
            const int row = row0 + 8 * b + 2 * t + e, i = row / a.group;
#pragma unroll
            for (int n = 0; n < 2; n++) {
              const int p = p0 + 16 * y + g + 8 * n;
              if (((held >> y) & 1u) && p < u.hi && row < u.rows && (p < u.sv.ctx || sees(a, u, i, p - u.sv.ctx)))
                seen[y] |= 1u << (4 * b + 2 * n + e);
            }
          }
      }
    }
    auto off = [&](int b, int y, int i) { return MASKED && !((seen[y] >> (4 * b + i)) & 1u); };
    float mx[NB][2];
    bool grow = false;
#pragma unroll
    for (int b = 0; b < NB; b++) {
#pragma unroll
      for (int e = 0; e < 2; e++) {
        float x = -CUDART_INF_F;
#pragma unroll
        for (int y = 0; y < TS; y++) {
          if (off(b, y, e)) s[b][y][e] = -CUDART_INF_F;
          if (off(b, y, 2 + e)) s[b][y][2 + e] = -CUDART_INF_F;
          x = fmaxf(x, fmaxf(s[b][y][e], s[b][y][2 + e]));
        }
        mx[b][e] = key_max(x) * rs[b][e];
        grow |= mx[b][e] > m[b][e] + GROW;  // m starts at -inf: a row's first position is always more
      }
    }
    if (__any_sync(0xffffffffu, grow)) {
#pragma unroll
      for (int b = 0; b < NB; b++)
#pragma unroll
        for (int e = 0; e < 2; e++) {
          if (!(mx[b][e] > m[b][e] + GROW)) continue;
          l[b][e] *= ex2(m[b][e] - mx[b][e]);
          // what o holds shrinks by the same factor, which goes into inv; past
          // 2^100 (at the first position, from infinity) into o
          const float f = inv[b][e] * ex2(mx[b][e] - m[b][e]);
          m[b][e] = mx[b][e];
          inv[b][e] = fminf(f, 0x1p100f);
          if (f > 0x1p100f) scale_row(b, e, 0x1p100f / f);
        }
    }
    float xm[NB][2];
    bool big = false;
#pragma unroll
    for (int b = 0; b < NB; b++)
#pragma unroll
      for (int e = 0; e < 2; e++) {
        const float mu = m[b][e] == -CUDART_INF_F ? 0.0f : m[b][e];
        float x = 0.0f;
#pragma unroll
        for (int y = 0; y < TS; y++)
#pragma unroll
          for (int n = 0; n < 2; n++) {
            const float p = ex2(fmaf(s[b][y][2 * n + e], rs[b][e], -mu));
            l[b][e] += p;
            s[b][y][2 * n + e] = off(b, y, 2 * n + e) ? 0.0f : p * dv[y][n];
            x = fmaxf(x, s[b][y][2 * n + e]);
          }
        xm[b][e] = x;
        big |= x * inv[b][e] > TOP;
      }
    if (__any_sync(0xffffffffu, big)) {
#pragma unroll
      for (int b = 0; b < NB; b++)
#pragma unroll
        for (int e = 0; e < 2; e++) {
          const float top = key_max(xm[b][e]);
          if (!(top * inv[b][e] > TOP)) continue;
          const float now = SET / fmaxf(top, 0x1p-100f);
          scale_row(b, e, now / inv[b][e]);
          inv[b][e] = now;
        }
    }
#pragma unroll
    for (int y = 0; y < TS; y++) {
      const uint32_t vb = sm + y * T::BYTES + T::CODES, vsc = vb + T::CODES + T::SCALES;
      uint32_t p[NT][NB][2];  // keys 2 t, 2 t + 1 (+ 8) of row 8 b + g
#pragma unroll
      for (int b = 0; b < NB; b++)
#pragma unroll
        for (int n = 0; n < 2; n++) {
          const float x0 = s[b][y][2 * n] * inv[b][0], x1 = s[b][y][2 * n + 1] * inv[b][1];
          const uint32_t hi = pack2(x0, x1);
          p[0][b][n] = transpose8(hi);
          if (NT == 2) p[NT - 1][b][n] = transpose8(rest2(x0, x1, hi));
        }
      // V: this lane's DH / 8 dimensions of keys 2 t, 2 t + 1, 2 t + 8, 2 t + 9
      constexpr int VB = RB / 8, VW = VB / 4;
      uint32_t v[2][2][VW];
      uint32_t sd[2] = {0, 0}, md[2] = {0, 0};
#pragma unroll
      for (int n = 0; n < 2; n++) {
#pragma unroll
        for (int e = 0; e < 2; e++) {
          const uint32_t at = vb + T::at(8 * n + 2 * t + e, g * VB);
          if (VB == 16) {
            const uint4 x = sld_v4(at);
            v[n][e][0] = x.x; v[n][e][1 % VW] = x.y; v[n][e][2 % VW] = x.z; v[n][e][3 % VW] = x.w;
          } else if (VB == 8) {
            const uint2 x = sld_v2(at);
            v[n][e][0] = x.x; v[n][e][1 % VW] = x.y;
          } else {
            v[n][e][0] = __float_as_uint(sld_f(at));
          }
        }
        if (TYPE == PK_KV_Q4) {
          const int sh = 4 * (g * (DH / 8) / 32);
          const uint4 x = sld_v4(vsc + (8 * n + 2 * t) * 8);  // D, sub, D, sub
          const int s0 = (int)((x.y >> sh) & 15u), s1 = (int)((x.w >> sh) & 15u);
          sd[n] = h2u(__halves2half2(__int2half_rn(s0), __int2half_rn(s1)));
          md[n] = h2u(__halves2half2(__int2half_rn(-1032 * s0), __int2half_rn(-1032 * s1)));
        }
      }
      // of a word's values two a product: dimensions d (rows 0-7), d + 1 (rows 8-15)
#pragma unroll
      for (int w = 0; w < VW; w++) {
        uint32_t x[2][2];
#pragma unroll
        for (int n = 0; n < 2; n++) {
          x[n][0] = __byte_perm(v[n][0][w], v[n][1][w], TYPE == PK_KV_Q8 ? 0x5140 : 0x5410);
          x[n][1] = __byte_perm(v[n][0][w], v[n][1][w], TYPE == PK_KV_Q8 ? 0x7362 : 0x7632);
        }
        constexpr int PW = TYPE == PK_KV_Q8 ? 2 : 4;  // products a word
#pragma unroll
        for (int d = 0; d < PW; d++) {
          uint32_t f[4];
#pragma unroll
          for (int n = 0; n < 2; n++)
#pragma unroll
            for (int e = 0; e < 2; e++) {
              if (TYPE == PK_KV_Q8) f[2 * n + e] = codes_of(x[n][d], e ? 0x4342 : 0x4140);
              else f[2 * n + e] = nibbles_of(x[n][d / 2] >> (4 * (2 * (d % 2) + e)), sd[n], md[n]);
            }
#pragma unroll
          for (int b = 0; b < NB; b++) {
            float(&acc)[4] = o[b][w * PW + d];
            if (NT == 2) {  // the tensor core's own sums drop bits below the running one's last; f32 adds round
              float c[4] = {0.0f, 0.0f, 0.0f, 0.0f};
              mma16816(c, f, p[NT - 1][b][0], p[NT - 1][b][1]);
              mma16816(c, f, p[0][b][0], p[0][b][1]);
#pragma unroll
              for (int i = 0; i < 4; i++) acc[i] += c[i];
            } else {
              mma16816(acc, f, p[0][b][0], p[0][b][1]);
            }
          }
        }
      }
    }
  }
};

// A CTA of 4 warps: RG groups of 8 NB rows times KG = 4 / RG groups of
// positions.  The warps of a key group share its ring of tiles; key group k
// takes every KG-th tile from k, and the groups are added up at the end.
constexpr int AW = 4;
template <int TYPE, int DH, int NT, int NB, int RG>
struct Geo {
  using T = Tile<TYPE, DH>;
  using W = Warp<TYPE, DH, NT, NB>;
  static constexpr int KG = AW / RG, ROWS = 8 * NB * RG;
  static constexpr int RING = KG * NSTAGE * T::BYTES;
  static constexpr int SUM = KG * ROWS * (DH + 4) * 4;  // outputs (rows padded by 16 bytes), then m, l, and theirs added up
  static constexpr int END = SUM + (KG + 1) * ROWS * 8;
  static constexpr int SMEM = RING + RG * W::QBYTES > END ? RING + RG * W::QBYTES : END;
};

template <int TYPE, int DH, int NT, int NB, int RG>
__global__ void __launch_bounds__(32 * AW) k_kv_attn(const AttnKArgs a) {
  using G = Geo<TYPE, DH, NT, NB, RG>;
  using T = typename G::T;
  extern __shared__ __align__(128) uint8_t smem[];
  pdl_trigger();
  pdl_wait();
  const Unit u = unit_of(a);
  const int tile0 = u.rt * G::ROWS;
  if (tile0 >= u.rows || (u.ch >= max(u.nch, 1) && !(a.cluster && u.nch > 1))) return;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, g = lane >> 2, t = lane & 3;
  const int rg = warp % RG, kg = warp / RG, row0 = tile0 + rg * 8 * NB;
  // without a mask nobody sees past the tile's last token
  const int last = (min(tile0 + G::ROWS, u.rows) - 1) / a.group;
  const int hi = a.q.mask ? u.hi : min(u.hi, u.sv.ctx + last + 1);
  // steps of TS tiles; key group k takes every KG-th step from k
  constexpr int TS = G::W::TS, PAIRS = NSTAGE / TS;
  const int span = hi - u.lo - 16 * TS * kg, nt = span > 0 ? (span + 16 * TS * G::KG - 1) / (16 * TS * G::KG) : 0;
  const uint32_t ring = shaddr(smem) + kg * NSTAGE * T::BYTES;
  const int ti = rg * 32 + lane, tn = 32 * RG;
  auto pos = [&](int i) { return u.lo + 16 * TS * (kg + G::KG * i); };
  // lane x holds the page of tile x of the block of 32 tiles being copied, and
  // of the one being used; -1: none
  auto pages_of = [&](int i0) {
    const int i = i0 + lane / TS, p = pos(i) + 16 * (lane % TS);
    if (i >= nt || p >= hi) return -1;
    const int j = p >> a.page_shift;
    const int pg = j < a.s.max_pages ? __ldg(a.s.pages + (size_t)u.s * a.s.max_pages + j) : -1;
    return pg >= 0 && pg < a.c.n_pages ? pg : -1;
  };
  constexpr int BLOCK = 32 / TS;  // steps
  int ahead = pages_of(0), now = ahead;
  auto issue = [&](int i) {
    if (i > 0 && i % BLOCK == 0) ahead = pages_of(i);
#pragma unroll
    for (int y = 0; y < TS; y++) {
      const int pg = __shfl_sync(0xffffffffu, ahead, (i % BLOCK) * TS + y);
      if (i < nt && pg >= 0) {
        const long long row = ((long long)pg * a.c.n_kv + u.h) * a.c.page_size + ((pos(i) + 16 * y) & (a.c.page_size - 1));
        T::copy(a.c, row, ring + ((i % PAIRS) * TS + y) * T::BYTES, ti, tn);
      }
    }
    cp_commit();
  };
#pragma unroll
  for (int i = 0; i < PAIRS - 1; i++) issue(i);
  typename G::W W;
  W.init(a, u, row0, lane, shaddr(smem) + G::RING + rg * G::W::QBYTES);
  __syncwarp();
  for (int i = 0; i < nt; i++) {
    cp_wait<PAIRS - 2>();
    if (RG > 1) bar_n(1 + kg, tn);
    else __syncwarp();
    if (i > 0 && i % BLOCK == 0) now = ahead;  // (the copies are less than a block ahead)
    uint32_t held = 0;
#pragma unroll
    for (int y = 0; y < TS; y++) held |= __shfl_sync(0xffffffffu, now, (i % BLOCK) * TS + y) >= 0 ? 1u << y : 0u;
    issue(i + PAIRS - 1);
    if (!held) continue;
    const uint32_t sm = ring + (i % PAIRS) * TS * T::BYTES;
    if (pos(i) + 16 * TS > min(u.sv.ctx, hi) || held != (1u << TS) - 1) W.template tile<true>(a, u, row0, pos(i), sm, held, lane);
    else W.template tile<false>(a, u, row0, pos(i), sm, held, lane);
  }
  cp_wait<0>();
  __syncthreads();  // the ring's memory is free
  float *so = reinterpret_cast<float *>(smem);
  float2 *sml = reinterpret_cast<float2 *>(smem + G::SUM), *sfin = sml + G::KG * G::ROWS;
#pragma unroll
  for (int b = 0; b < NB; b++)
#pragma unroll
    for (int e = 0; e < 2; e++) {
      float l = W.l[b][e];
      l += __shfl_xor_sync(0xffffffffu, l, 4);
      l += __shfl_xor_sync(0xffffffffu, l, 8);
      l += __shfl_xor_sync(0xffffffffu, l, 16);
      const int r = kg * G::ROWS + rg * 8 * NB + 8 * b + 2 * t + e;
      if (g == 0) sml[r] = make_float2(W.m[b][e], l);
      const float f = 1.0f / W.inv[b][e];
#pragma unroll
      for (int i = 0; i < DH / 16; i += 2)
        *reinterpret_cast<float4 *>(so + r * (DH + 4) + g * (DH / 8) + 2 * i) =
            make_float4(W.o[b][i][e] * f, W.o[b][i][2 + e] * f, W.o[b][i + 1][e] * f, W.o[b][i + 1][2 + e] * f);
    }
  __syncthreads();
  const bool cluster = a.cluster && u.nch > 1;
  for (int x = threadIdx.x; x < G::ROWS * 8; x += 32 * AW) {
    const int r = x >> 3, d0 = (x & 7) * (DH / 8);
    if (tile0 + r >= u.rows) continue;
    float M = -CUDART_INF_F, L = 0.0f, acc[DH / 8];
#pragma unroll
    for (int k = 0; k < G::KG; k++) M = fmaxf(M, sml[k * G::ROWS + r].x);
#pragma unroll
    for (int j = 0; j < DH / 8; j++) acc[j] = 0.0f;
#pragma unroll
    for (int k = 0; k < G::KG; k++) {
      const float2 ml = sml[k * G::ROWS + r];
      const float f = ml.y == 0.0f ? 0.0f : ex2(ml.x - M);  // a NaN sum stays one
      L = fmaf(f, ml.y, L);
#pragma unroll
      for (int j = 0; j < DH / 8; j++) acc[j] = fmaf(f, so[(k * G::ROWS + r) * (DH + 4) + d0 + j], acc[j]);
    }
    if (cluster) {  // in the place of the first group's
#pragma unroll
      for (int j = 0; j < DH / 8; j++) so[r * (DH + 4) + d0 + j] = acc[j];
      if (d0 == 0) sfin[r] = make_float2(M, L);
      continue;
    }
    if (u.nch > 1) {
      if (d0 == 0) {
        const int i = (tile0 + r) / a.group, h = u.h * a.group + (tile0 + r) - i * a.group;
        a.part_ml[((long long)(u.sv.first + i) * a.q.n_head + h) * a.n_chunk + u.ch] = make_float2(M, L);
      }
    } else {
      const float inv = L > 0.0f || isnan(L) ? 1.0f / L : 0.0f;
#pragma unroll
      for (int j = 0; j < DH / 8; j++) acc[j] *= inv;
    }
    write_row<DH>(a, u, tile0 + r, d0, acc, u.nch > 1);
  }
  if (cluster) join_cluster<DH>(a, u, tile0, G::ROWS, shaddr(so), shaddr(sfin), 32 * AW);
}

// Adds up the chunks of rows that have more than one.  W warps a row, each with
// every W-th chunk, four chunks' loads at a time: 1 (four rows a CTA) where
// there are up to 8 chunks, 8 where there are more (one sequence of 30000
// positions has 118, which one warp took longer over than the attention).
template <int DH, int W>
__global__ void __launch_bounds__(W == 1 ? 128 : 32 * W) k_kv_attn_join(const AttnKArgs a) {
  constexpr int V = DH / 32;
  __shared__ float so[W][DH];
  __shared__ float2 sml[W];
  pdl_trigger();
  pdl_wait();
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const long long row = W == 1 ? (long long)blockIdx.x * 4 + warp : (long long)blockIdx.x;
  const long long tok = row / a.q.n_head;
  const int h = (int)(row - tok * a.q.n_head), w = W == 1 ? 0 : warp;
  if (tok >= a.s.n_tok) return;  // (whole warps; with W > 1 the whole CTA, as all returns here)
  const int s = seq_of(a.s, (int)tok, lane);
  if (s < 0) return;
  const SeqView sv = seq_view(a.s, a.c.page_size, s);
  const int nch = (sv.total + a.chunk - 1) / a.chunk;
  if (tok - sv.first >= sv.n || nch <= 1) return;
  const float2 *ml = a.part_ml + row * a.n_chunk;
  const float *po = a.part_o + row * a.n_chunk * DH + V * lane;
  float M = -CUDART_INF_F;
  for (int c = w + W * lane; c < nch; c += 32 * W) M = fmaxf(M, ml[c].x);
#pragma unroll
  for (int i = 16; i > 0; i >>= 1) M = fmaxf(M, __shfl_xor_sync(0xffffffffu, M, i));
  float L = 0.0f, acc[V];
#pragma unroll
  for (int j = 0; j < V; j++) acc[j] = 0.0f;
  for (int c0 = w; c0 < nch; c0 += 4 * W) {
    float2 x[4];
    float v[4][V];
#pragma unroll
    for (int k = 0; k < 4; k++) {
      const int c = min(c0 + k * W, nch - 1);
      x[k] = ml[c];
      if (V == 4) *reinterpret_cast<float4 *>(v[k]) = *reinterpret_cast<const float4 *>(po + (size_t)c * DH);
      else *reinterpret_cast<float2 *>(v[k]) = *reinterpret_cast<const float2 *>(po + (size_t)c * DH);
    }
#pragma unroll
    for (int k = 0; k < 4; k++) {
      const float f = c0 + k * W >= nch || x[k].y == 0.0f ? 0.0f : ex2(x[k].x - M);  // a NaN sum stays one
      L = fmaf(f, x[k].y, L);
#pragma unroll
      for (int j = 0; j < V; j++)
        if (f != 0.0f) acc[j] = fmaf(f, v[k][j], acc[j]);
    }
  }
  if (W > 1) {
    if (lane == 0) sml[w] = make_float2(M, L);
#pragma unroll
    for (int j = 0; j < V; j++) so[w][V * lane + j] = acc[j];
    __syncthreads();
    if (w > 0) return;
    M = -CUDART_INF_F;
#pragma unroll
    for (int k = 0; k < W; k++) M = fmaxf(M, sml[k].x);
    L = 0.0f;
#pragma unroll
    for (int j = 0; j < V; j++) acc[j] = 0.0f;
#pragma unroll
    for (int k = 0; k < W; k++) {
      const float f = sml[k].y == 0.0f ? 0.0f : ex2(sml[k].x - M);
      L = fmaf(f, sml[k].y, L);
#pragma unroll
      for (int j = 0; j < V; j++) acc[j] = fmaf(f, so[k][V * lane + j], acc[j]);
    }
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

// The kernel's variant by the rows that a kv head's tile may have: columns in
// steps of 8 up to 32 a warp (16 where f32's two terms double the query
// fragments of 128 dimensions), then two or four warps side by side.
struct Variant {
  void (*k)(AttnKArgs) = nullptr;
  int smem = 0, rows = 0;
};
template <int TYPE, int DH, int NT, int NB, int RG>
Variant variant_as() {
  using G = Geo<TYPE, DH, NT, NB, RG>;
  return {k_kv_attn<TYPE, DH, NT, NB, RG>, G::SMEM, G::ROWS};
}
// From TC_FROM rows on half-precision queries take the tcgen05 kernel, whose
// time hardly depends on the rows up to 128 (40 sequences of 7500 and 15000
// positions, Q4: 16 rows 252 us here and 340 there, 8 rows 188 and 337; past 16
// a row tile here takes twice as long), f32 ones of head_dim 64 from TC32_FROM
// (8 sequences of 2000 positions, 36 heads: 32 rows 91 us here; 33 rows 138 and
// 111; 128 rows 253 and 130).
constexpr long long TC_FROM = 17, TC32_FROM = 33;
template <int TYPE, int DH, int NT>
Variant variant_rows(long long rows) {
  if (rows <= 8) return variant_as<TYPE, DH, NT, 1, 1>();
  if (rows <= 16) return variant_as<TYPE, DH, NT, 2, 1>();
  if constexpr (NT == 1) {
    static_assert(TC_FROM == 17, "half-precision rows past 16");
    return {nullptr, 0, 128};
  } else if constexpr (DH == 64) {
    static_assert(TC32_FROM == 33, "f32 rows past 32");
    return rows <= 32 ? variant_as<TYPE, DH, NT, 4, 1>() : Variant{nullptr, 0, 256};
  } else {
    return rows <= 32 ? variant_as<TYPE, DH, NT, 2, 2>() : variant_as<TYPE, DH, NT, 2, 4>();
  }
}
template <int TYPE, int DH>
Variant variant_type(int type, long long rows) {
  return type == T_F32 ? variant_rows<TYPE, DH, 2>(rows) : variant_rows<TYPE, DH, 1>(rows);
}
Variant variant_of(const pk_kv_cache &c, const pk_kv_seqs &s, int n_head, int type) {
  const long long rows = (long long)s.max_new * (n_head / c.n_kv);
  if (c.type == PK_KV_Q8) return c.head_dim == 64 ? variant_type<PK_KV_Q8, 64>(type, rows) : variant_type<PK_KV_Q8, 128>(type, rows);
  return c.head_dim == 64 ? variant_type<PK_KV_Q4, 64>(type, rows) : variant_type<PK_KV_Q4, 128>(type, rows);
}

// Chunks of a sequence's positions: so many that 148 SMs have about eight CTAs
// each, none under MIN_CHUNK positions.  Where all CTAs run at once (two an SM)
// up to eight chunks are a cluster, whose CTAs add up through one another's
// shared memory (up to 16 are made 8): that saves the scratch and a second
// launch, 13 us to 11 for one token at 1500 positions.  Elsewhere a cluster's
// CTAs would hold their SMs until its longest is done (eight 16K streams 171 us
// against 150), so their parts go through the scratch.  The tcgen05 kernel's chunks
// are as many as take the least time by its rounds of CTAs: a CTA costs its
// tiles of 64 positions and 16 more (one CTA an SM: 8) for its beginning and
// its part of the sums, and where two share an SM a tile takes 8 fifths of what
// it takes alone (64 tokens at 8000 positions, 64 heads over 8: 4 chunks, one
// CTA an SM, 53 us, 8 chunks 66, one 127, 37 100; 32 sequences of 2000: one
// chunk 61, two 79, four 100; the wide trees 770, 799 and 750, one and four of
// which this estimates within 1% of each other).
struct Split {
  int chunk, n_chunk, row_tiles;
  bool cluster;
  bool parts;  // partial results go through the scratch
};
Split split_of(const pk_kv_cache &c, const pk_kv_seqs &s, int n_head, int type, const Variant &v) {
  Split p;
  const long long rows = (long long)s.max_new * (n_head / c.n_kv);
  p.row_tiles = (int)((rows + v.rows - 1) / v.rows);
  const long long units = (long long)s.n_seq * c.n_kv * p.row_tiles, want = 148 * 8;
  const long long most = (s.max_len + MIN_CHUNK - 1) / MIN_CHUNK;
  const long long sum = sum_most(type), least = v.k && type != T_F32 ? (s.max_len + 4 * sum - 1) / (4 * sum) : 1;
  long long n = std::max(least, std::min(most, want / units));
  if (!v.k) {
    long long best = 0;
    const long long top = n;
    for (long long c = 1; c <= top; c++) {
      const long long ctas = units * c, left = ctas % 296, tiles = ((s.max_len + 63) / 64 + c - 1) / c;
      const long long t = v.rows == 256 ? (ctas + 147) / 148 * (tiles + 8)
                                        : (ctas / 296 * 8 + (left == 0 ? 0 : left <= 148 ? 5 : 8)) * (tiles + 16);
      if (c == 1 || t < best) best = t, n = c;
    }
  }
  const long long slots = v.rows == 256 ? 128 : 296;  // CTAs that run at once, in clusters too
  if (v.k && n > 8 && n <= 16 && least <= 8 && units * 8 <= slots) n = 8;
  p.chunk = (int)(((s.max_len + n - 1) / n + 63) / 64 * 64);
  p.n_chunk = (int)((s.max_len + (long long)p.chunk - 1) / p.chunk);
  p.cluster = p.n_chunk > 1 && p.n_chunk <= 8 && units * p.n_chunk <= slots;
  p.parts = (p.n_chunk > 1 && !p.cluster) || (!v.k && type != T_F32 && p.chunk > sum);
  return p;
}

}  // namespace

// max_new and max_len are the caller's bounds and may be any numbers; no
// sequence has more new tokens than there are, or more positions than its pages
// hold, which the kernel, the grid and the scratch go by.
static pk_kv_seqs bounded(const pk_kv_cache &c, pk_kv_seqs s) {
  s.max_new = std::min(s.max_new, s.n_tok);
  s.max_len = (int)std::min<long long>(s.max_len, (long long)s.max_pages * c.page_size);
  return s;
}

size_t kv_attn_scratch_bytes(const pk_kv_cache &c, const pk_kv_seqs &seqs, int n_head, int type) {
  const pk_kv_seqs s = bounded(c, seqs);
  const Split p = split_of(c, s, n_head, type, variant_of(c, s, n_head, type));
  if (!p.parts) return 0;
  return (size_t)s.n_tok * n_head * p.n_chunk * (c.head_dim + 2) * sizeof(float);
}

bool kv_attn_waits(const pk_kv_cache &c, const pk_kv_seqs &seqs, int n_head, int type) {
  return !variant_of(c, bounded(c, seqs), n_head, type).k;
}

cudaError_t launch_kv_attn(const pk_kv_cache &c, const pk_kv_seqs &seqs, const pk_kv_query &q, void *scratch,
                           cudaStream_t st, int *err, bool poison) {
  const pk_kv_seqs s = bounded(c, seqs);
  const Variant v = variant_of(c, s, q.n_head, q.type);
  const Split p = split_of(c, s, q.n_head, q.type, v);
  AttnKArgs a{};
  a.c = c; a.s = s; a.q = q;
  a.chunk = p.chunk; a.n_chunk = p.n_chunk; a.row_tiles = p.row_tiles;
  a.group = q.n_head / c.n_kv;
  while ((1 << a.page_shift) < c.page_size) a.page_shift++;
  const uintptr_t es = q.type == T_F32 ? 4 : 2;
  a.vec_q = (((uintptr_t)q.q | (uintptr_t)q.q_tok_stride * es | (uintptr_t)q.q_head_stride * es) & 15) == 0;
  a.vec_o = (((uintptr_t)q.out | (uintptr_t)q.out_tok_stride * es | (uintptr_t)q.out_head_stride * es) & 15) == 0;
  const size_t rows = (size_t)s.n_tok * q.n_head;
  a.part_o = reinterpret_cast<float *>(scratch);
  a.cluster = p.cluster;
  a.err = err;
  a.poison = poison;
  a.part_ml = p.parts ? reinterpret_cast<float2 *>(a.part_o + rows * p.n_chunk * c.head_dim) : nullptr;
  const long long blocks = (long long)s.n_seq * c.n_kv * p.row_tiles * p.n_chunk, jb = ((long long)rows + 3) / 4;
  if (blocks > 0x7fffffffLL || (long long)rows > 0x7fffffffLL) return cudaErrorInvalidValue;
  const int cluster = a.cluster ? p.n_chunk : 1;
  cudaError_t e;
  if (!v.k) e = launch_kv_attn_tc(a, cluster, (unsigned)blocks, st);
  else e = launch_cluster(v.k, cluster, dim3((unsigned)blocks), dim3(32 * AW), v.smem, st, a);
  if (e != cudaSuccess || p.n_chunk <= 1 || a.cluster) return e;
  if (p.n_chunk <= 8) return launch(c.head_dim == 64 ? k_kv_attn_join<64, 1> : k_kv_attn_join<128, 1>, dim3((unsigned)jb), dim3(128), 0, st, a);
  return launch(c.head_dim == 64 ? k_kv_attn_join<64, 8> : k_kv_attn_join<128, 8>, dim3((unsigned)rows), dim3(256), 0, st, a);
}

}  // namespace pk
