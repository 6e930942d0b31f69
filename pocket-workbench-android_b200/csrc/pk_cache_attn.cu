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

// SHARED: calls over shared prefixes, a form of its own, as the registers that
// joining takes cost others CTAs (104 and 176 a thread for 96 and 140 with 8 f32 rows
// of 64 and of 128 dimensions).
template <int TYPE, int DH, int NT, int NB, int RG, bool SHARED>
__global__ void __launch_bounds__(32 * AW) k_kv_attn(const AttnKArgs a) {
  using G = Geo<TYPE, DH, NT, NB, RG>;
  using T = typename G::T;
  extern __shared__ __align__(128) uint8_t smem[];
  // (a prefixes' launch has all work before it behind it as it begins, and so has the
  // launch that it lets begin; its wait, for nothing, in one place with the others'
  // takes a register more: 12 groups 74 us for 68)
  if (SHARED && a.mode == ATTN_PREFIX) pdl_wait();
  pdl_trigger();
  if (!SHARED || (a.mode != ATTN_PREFIX && !a.early)) pdl_wait();
  const Unit u = unit_of<SHARED>(a);
  const int tile0 = u.rt * G::ROWS;
  if (idle<SHARED>(a, u, tile0)) {
    if (SHARED) end_early(a);
    return;
  }
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
  if (SHARED && a.merge && a.early) pdl_wait();
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
    if (u.part) {
      if (d0 == 0) {
        const int i = (tile0 + r) / a.group, h = u.h * a.group + (tile0 + r) - i * a.group;
        a.part_ml[((long long)(u.sv.first + i) * a.q.n_head + h) * a.n_part + u.slot] = make_float2(M, L);
      }
    } else if (SHARED && a.merge) {
      merge_in<DH / 8>(merge_of<DH>(a, u, tile0 + r, M, L), DH, d0, acc);
    } else {
      const float inv = L > 0.0f || isnan(L) ? 1.0f / L : 0.0f;
#pragma unroll
      for (int j = 0; j < DH / 8; j++) acc[j] *= inv;
    }
    write_row<DH>(a, u, tile0 + r, d0, acc, u.part);
  }
  if (SHARED && !a.merge) end_early(a);
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
  int nch = (sv.total + a.chunk - 1) / a.chunk, npre = 0;
  if (tok - sv.first >= sv.n) return;
  if (a.mode == ATTN_OWN) {
    const OwnView v = own_view(a, s, sv);
    npre = (v.base + a.pre_chunk - 1) / a.pre_chunk;
    nch = npre + (v.total - v.base + a.chunk - 1) / a.chunk;
  } else if (nch <= 1) {
    return;
  }
  // (parts npre .. are the row's own, which lie from n_pre on)
  const float2 *ml = a.part_ml + row * a.n_part;
  const float *po = a.part_o + row * a.n_part * DH + V * lane;
  auto at = [&](int c) { return c < npre ? c : c - npre + a.n_pre; };
  float M = -CUDART_INF_F;
  for (int c = w + W * lane; c < nch; c += 32 * W) M = fmaxf(M, ml[at(c)].x);
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
      const int c = at(min(c0 + k * W, nch - 1));
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

// The tcgen05 kernel's time for so many CTAs of so many tiles of 64 positions, by
// rounds: a tile's time, and as many tiles more for a CTA's beginning and its part of
// the sums.  Half precision, in proportions: 16 tiles more, and where two CTAs share
// an SM a tile takes 8 fifths of what it takes alone (64 tokens at 8000 positions, 64
// heads over 8: 4 chunks, one CTA an SM, 53 us, 8 chunks 66, one 127, 37 100; 32
// sequences of 2000: one chunk 61, two 79, four 100; wide trees 770, 799 and 750, one
// and four of which this estimates within 1% of each other).  f32 (head_dim 64), in
// 100 ns: CTAs of two blocks, one an SM, 1.3 us and 11 tiles (36 heads, 64 tokens of a
// sequence at 8000: one chunk 182 us, two 98, four 60); of one block, 1.5 and 14 where
// it has the SM to itself (one chunk 216, two 119), 2.0 and 9 where two share it (8
// sequences with 33 tokens, at 2000 82, at 16000 529; 40 of 200, 16 heads, 67).
long long tc_time(int type, int rows, long long ctas, long long tiles) {
  if (rows == 256) return (ctas + 147) / 148 * 13 * (tiles + 11);
  const long long rounds = ctas / 296, left = ctas % 296;
  const bool one = left > 0 && left <= 148, two = left > 148;
  if (type == T_F32) return (rounds + two) * 20 * (tiles + 9) + one * 15 * (tiles + 14);
  return (rounds * 8 + (one ? 5 : two ? 8 : 0)) * (tiles + 16);
}
// The chunks of the least time, up to `top` and from one on.  Not those of f32 in
// clusters that do not all run at once: of CTAs of one block 148 SMs have room for 296
// alone or in pairs, for 259 in clusters of seven; of two blocks for 130 and more, but
// 105 in clusters of seven and 120 of eight (a sequence of 8000, 36 heads, 64 tokens:
// 6 chunks 61 us, 8 88; of 3712, 16 heads, 43 tokens, two blocks: 8 48, 9 25).
long long tc_chunks(int type, int rows, long long units, int max_len, long long top, bool parts, long long *time = nullptr) {
  long long n = 1, best = 0;
  for (long long c = 1; c <= top; c++) {
    const long long ctas = units * c;
    const bool cluster = !parts && c > 1 && c <= 8 && ctas <= (rows == 256 ? 128 : 296);
    if (type == T_F32 && cluster && c > 2 && ctas > (rows == 128 ? 256 : c < 7 ? 128 : 105)) continue;
    long long t = tc_time(type, rows, ctas, ((max_len + 63LL) / 64 + c - 1) / c);
    if (type == T_F32 && !parts && c > 1 && !cluster) t += 25;  // (a launch that joins)
    if (c == 1 || t < best) best = t, n = c;
  }
  if (time) *time = best;
  return n;
}
constexpr long long WANT = 148 * 8;  // CTAs
// Chunks there may be: WANT CTAs, none under MIN_CHUNK positions.
long long most_chunks(long long units, int max_len) { return std::max(1LL, std::min((max_len + MIN_CHUNK - 1LL) / MIN_CHUNK, WANT / units)); }

// The kernel's variant by the rows that a kv head's tile may have: columns in
// steps of 8 up to 32 a warp (16 where f32's two terms double the query
// fragments of 128 dimensions), then two or four warps side by side.
struct Variant {
  void (*k)(AttnKArgs) = nullptr, (*shared)(AttnKArgs) = nullptr;
  int smem = 0, rows = 0;
};
template <int TYPE, int DH, int NT, int NB, int RG>
Variant variant_as() {
  using G = Geo<TYPE, DH, NT, NB, RG>;
  // Eight half-precision rows of 64 Q8 codes: four CTAs an SM by their shared memory,
  // where registers allow five and 148 SMs then have the eight that each gets in one
  // round and part of another (36 heads: 8 streams of 16256 121 us with five, 109 with
  // four, 16 of 16000 224 and 199, one of 4000 12.7 and 11.7; 4 kv heads: 8 of 4000
  // 13.5 and 12.3, 16 of 16000 37.3 and 38.9).  In 4 bits five are no slower.
  constexpr bool FOUR = TYPE == PK_KV_Q8 && DH == 64 && NT == 1 && NB == 1;
  constexpr int SMEM = FOUR && G::SMEM < 48 * 1024 ? 48 * 1024 : G::SMEM;
  return {k_kv_attn<TYPE, DH, NT, NB, RG, false>, k_kv_attn<TYPE, DH, NT, NB, RG, true>, SMEM, G::ROWS};
}
// From TC_FROM rows on half-precision queries take the tcgen05 kernel, whose
// time hardly depends on the rows up to 128 (40 sequences of 7500 and 15000
// positions, Q4: 16 rows 252 us here and 340 there, 8 rows 188 and 337; past 16
// a row tile here takes twice as long), f32 ones of head_dim 64 from TC32_FROM
// (8 sequences of 2000 positions, 36 heads: 32 rows 91 us here, 33 rows 138 here and
// 84 there, 128 rows 253 and 95; of 16000 positions 32 rows 367 here, 33 529 there).
constexpr long long TC_FROM = 17, TC32_FROM = 33;
template <int TYPE, int DH, int NT>
Variant variant_rows(long long rows) {
  if (rows <= 8) return variant_as<TYPE, DH, NT, 1, 1>();
  if (rows <= 16) return variant_as<TYPE, DH, NT, 2, 1>();
  if constexpr (NT == 1) {
    static_assert(TC_FROM == 17, "half-precision rows past 16");
    return {nullptr, nullptr, 0, 128};
  } else if constexpr (DH == 64) {
    static_assert(TC32_FROM == 33, "f32 rows past 32");
    return rows <= 32 ? variant_as<TYPE, DH, NT, 4, 1>() : Variant{nullptr, nullptr, 0, rows <= 128 ? 128 : 256};
  } else {
    return rows <= 32 ? variant_as<TYPE, DH, NT, 2, 2>() : variant_as<TYPE, DH, NT, 2, 4>();
  }
}
template <int TYPE, int DH>
Variant variant_type(int type, long long rows) {
  return type == T_F32 ? variant_rows<TYPE, DH, 2>(rows) : variant_rows<TYPE, DH, 1>(rows);
}
// tiles_too: more than 8 rows may go a tile of 8 at a time, each reading the cache
// again (from L2), where that is less work.  Against the tcgen05 kernel, a CTA of
// which costs its tiles of 64 positions and 16 more for its beginning and end, one
// here costs 4 more; its tile takes 10 eighteenths of the time there, and 10
// thirty-sixths where CTAs are so few that only their latency counts.  Against
// wider tiles here it is better in the second case, where there is little to do:
// code for 16 rows a warp is twice as long, and a CTA of few tiles waits for
// instructions most of its time.  (96 sequences of 24 rows and up to 318 positions behind 12
// prefixes: the call 69 us so, 91 with tiles of 16, 108 with the tcgen05 kernel; 4
// answers to a prompt of 700: 12, 17 and 31.)
Variant variant_of(const pk_kv_cache &c, const pk_kv_seqs &s, int n_head, int type, bool tiles_too = false) {
  long long rows = (long long)s.max_new * (n_head / c.n_kv);
  if (tiles_too && rows > 8) {
    const long long tiles = (s.max_len + 63) / 64, each = (rows + 7) / 8;
    const bool few = (long long)s.n_seq * c.n_kv * each <= 148, tc = rows >= (type != T_F32 ? TC_FROM : c.head_dim == 64 ? TC32_FROM : 1LL << 40);
    if (tc ? each * (tiles + 4) * 10 < (rows + 127) / 128 * (tiles + 16) * (few ? 36 : 18) : few && each * tiles <= 256) rows = 8;
  }
  Variant v = c.type == PK_KV_Q8 ? c.head_dim == 64 ? variant_type<PK_KV_Q8, 64>(type, rows) : variant_type<PK_KV_Q8, 128>(type, rows)
                                 : c.head_dim == 64 ? variant_type<PK_KV_Q4, 64>(type, rows) : variant_type<PK_KV_Q4, 128>(type, rows);
  // f32 rows that one block holds: in CTAs of one block, two an SM, or in CTAs of two,
  // one of them without rows, one an SM, which are done sooner where CTAs are few
  // (36 heads; one block and two: 64 tokens of a sequence at 8000 61 and 60 us, 128
  // at 4000 47 and 43, 4 sequences of 1000 with 128 45 and 43; 3 of 2000 with 33 49 and
  // 57, 8 of them with 64 87 and 119, 4 of 16000 with 128 284 and 359; 40 of 183 with
  // 35, 16 heads, 67 and 96).  Estimates within a twentieth count as equal.
  if (!v.k && type == T_F32 && v.rows == 128 && !tiles_too) {
    const long long units = (long long)s.n_seq * c.n_kv, top = most_chunks(units, s.max_len);
    long long one = 0, two = 0;
    tc_chunks(type, 128, units, s.max_len, top, false, &one);
    tc_chunks(type, 256, units, s.max_len, top, false, &two);
    if (two * 20 <= one * 21) v.rows = 256;
  }
  return v;
}

// Chunks of a sequence's positions: so many that 148 SMs have about eight CTAs
// each, none under MIN_CHUNK positions.  Where all CTAs run at once (two an SM)
// up to eight chunks are a cluster, whose CTAs add up through one another's
// shared memory (up to 16 are made 8): that saves the scratch and a second
// launch, 13 us to 11 for one token at 1500 positions.  Elsewhere a cluster's
// CTAs would hold their SMs until its longest is done (eight 16K streams 171 us
// against 150), so their parts go through the scratch.  The tcgen05 kernel's chunks
// are as many as take the least time by tc_time.
struct Split {
  int chunk, n_chunk, row_tiles;
  bool cluster;
  bool parts;  // partial results go through the scratch
};
// parts: through the scratch in any case.
Split split_of(const pk_kv_cache &c, const pk_kv_seqs &s, int n_head, int type, const Variant &v, bool parts = false) {
  Split p;
  const long long rows = (long long)s.max_new * (n_head / c.n_kv);
  p.row_tiles = (int)((rows + v.rows - 1) / v.rows);
  const long long units = (long long)s.n_seq * c.n_kv * p.row_tiles;
  const long long sum = sum_most(type), least = v.k && type != T_F32 ? (s.max_len + 4 * sum - 1) / (4 * sum) : 1;
  long long n = std::max(least, most_chunks(units, s.max_len));
  if (!v.k) n = tc_chunks(type, v.rows, units, s.max_len, n, parts);
  const long long slots = v.rows == 256 ? 128 : 296;  // CTAs that run at once, in clusters too
  if (!parts && v.k && n > 8 && n <= 16 && least <= 8 && units * 8 <= slots) n = 8;
  p.chunk = (int)(((s.max_len + n - 1) / n + 63) / 64 * 64);
  p.n_chunk = (int)((s.max_len + (long long)p.chunk - 1) / p.chunk);
  p.cluster = !parts && p.n_chunk > 1 && p.n_chunk <= 8 && units * p.n_chunk <= slots;
  p.parts = parts || (p.n_chunk > 1 && !p.cluster) || (!v.k && type != T_F32 && p.chunk > sum);
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

// What the launches of a call share.
static AttnKArgs args_of(const pk_kv_cache &c, const pk_kv_seqs &s, const pk_kv_query &q) {
  AttnKArgs a{};
  a.c = c; a.s = s; a.q = q;
  a.group = q.n_head / c.n_kv;
  while ((1 << a.page_shift) < c.page_size) a.page_shift++;
  const uintptr_t es = q.type == T_F32 ? 4 : 2;
  a.vec_q = (((uintptr_t)q.q | (uintptr_t)q.q_tok_stride * es | (uintptr_t)q.q_head_stride * es) & 15) == 0;
  a.vec_o = (((uintptr_t)q.out | (uintptr_t)q.out_tok_stride * es | (uintptr_t)q.out_head_stride * es) & 15) == 0;
  return a;
}
// units: sequences, or groups of them.
static cudaError_t launch_parts(AttnKArgs &a, const Variant &v, const Split &p, int units, cudaStream_t st) {
  a.chunk = p.chunk; a.n_chunk = p.n_chunk; a.row_tiles = p.row_tiles;
  a.cluster = p.cluster;
  const long long blocks = (long long)units * a.c.n_kv * p.row_tiles * p.n_chunk;
  if (blocks > 0x7fffffffLL) return cudaErrorInvalidValue;
  const int cluster = a.cluster ? p.n_chunk : 1;
  if (!v.k) return launch_kv_attn_tc(a, v.rows, cluster, (unsigned)blocks, st);
  return launch_as(a.mode != ATTN_PREFIX, a.mode == ATTN_ALL ? v.k : v.shared, cluster, dim3((unsigned)blocks), dim3(32 * AW), v.smem, st, a);
}
static cudaError_t launch_join(const AttnKArgs &a, cudaStream_t st) {
  const size_t rows = (size_t)a.s.n_tok * a.q.n_head;
  if (a.n_part <= 8)
    return launch(a.c.head_dim == 64 ? k_kv_attn_join<64, 1> : k_kv_attn_join<128, 1>, dim3((unsigned)((rows + 3) / 4)), dim3(128), 0, st, a);
  return launch(a.c.head_dim == 64 ? k_kv_attn_join<64, 8> : k_kv_attn_join<128, 8>, dim3((unsigned)rows), dim3(256), 0, st, a);
}

cudaError_t launch_kv_attn(const pk_kv_cache &c, const pk_kv_seqs &seqs, const pk_kv_query &q, void *scratch,
                           cudaStream_t st, int *err, bool poison) {
  const pk_kv_seqs s = bounded(c, seqs);
  const Variant v = variant_of(c, s, q.n_head, q.type);
  const Split p = split_of(c, s, q.n_head, q.type, v);
  AttnKArgs a = args_of(c, s, q);
  const size_t rows = (size_t)s.n_tok * q.n_head;
  if (rows > 0x7fffffff) return cudaErrorInvalidValue;
  a.n_part = p.n_chunk;
  a.part_o = reinterpret_cast<float *>(scratch);
  a.part_ml = p.parts ? reinterpret_cast<float2 *>(a.part_o + rows * p.n_chunk * c.head_dim) : nullptr;
  a.err = err;
  a.poison = poison;
  const cudaError_t e = launch_parts(a, v, p, s.n_seq, st);
  return e != cudaSuccess || p.n_chunk <= 1 || a.cluster ? e : launch_join(a, st);
}

// Shared prefixes: the groups as sequences of their tokens over the positions
// that they share, then each sequence over the rest of its own.  The second launch
// begins beside the first one's last CTAs (it reads nothing that the first one
// writes until it joins).  What it reads before it waits (lengths, tables, queries,
// the cache) earlier work may have written: the first launch is therefore not
// programmatic, so that in the stream's order all of that work is done and its
// writes are in memory before the first launch begins, and the second begins after
// it.  (Both programmatic: as long in a graph, four answers to a prompt 10.9 us and
// 11.0, 64 streams 47.4 and 46.7, and 1 to 2 us less called from a stream, 48.9 and
// 49.7; a second launch that waits first: 15.6 and 50.4.)  It adds the prefix's parts to its rows itself where a
// sequence's rest is one chunk; otherwise a third one joins all parts.  64 streams
// behind 4001 positions: 48 us, 17 less than with three launches one after another;
// every stream by itself over all its positions 101.
namespace {
struct Shared {
  pk_kv_seqs pre, own;  // bounds of the two
  Variant pre_v, own_v;
  Split pre_p, own_p;
  bool wide;   // the first is pk_cache_prefix.cu's
  bool merge;  // the second launch joins
};
Shared shared_plan(const pk_kv_cache &c, const pk_kv_seqs &s, const pk_kv_shared &sh, int n_head, int type) {
  Shared x;
  x.pre = x.own = s;
  x.pre.n_seq = sh.n_group;
  x.pre.max_new = std::min(sh.max_tok, s.n_tok);
  x.pre.max_len = std::min(sh.max_len, s.max_len) & ~15;
  // (and up to 15 of a shared length that is no multiple of 16)
  x.own.max_len = (int)std::min((long long)sh.max_own + 15, (long long)s.max_len);
  x.pre_p = x.own_p = Split{};
  x.wide = x.merge = false;
  if (x.pre.n_seq > 0 && x.pre.max_new > 0 && x.pre.max_len > 0) {
    x.pre_v = variant_of(c, x.pre, n_head, type, true);
    x.pre_p = split_of(c, x.pre, n_head, type, x.pre_v, true);
    // Half precision with more than a block of 128 rows: chunks by the rounds of
    // CTAs that they take, one an SM, at a CTA's tiles of 128 positions and 10 more.
    const long long rows = (long long)x.pre.max_new * (n_head / c.n_kv);
    x.wide = type != T_F32 && rows > 128;
    if (x.wide) {
      x.pre_p.row_tiles = (int)((rows + PREFIX_ROWS - 1) / PREFIX_ROWS);
      const long long units = (long long)sh.n_group * c.n_kv * x.pre_p.row_tiles, all = (x.pre.max_len + 127) / 128;
      const long long least = (x.pre.max_len + sum_most(type) - 1) / sum_most(type), most = std::max<long long>(least, MERGE);
      long long n = least, best = 0;
      for (long long k = least; k <= std::min(all, most); k++) {
        const long long t = (units * k + 147) / 148 * ((all + k - 1) / k + 10);
        if (k == least || t < best) best = t, n = k;
      }
      x.pre_p.chunk = (int)((all + n - 1) / n * 128);
      x.pre_p.n_chunk = (int)((x.pre.max_len + (long long)x.pre_p.chunk - 1) / x.pre_p.chunk);
    }
  }
  if (x.own.max_len > 0) {
    x.own_v = variant_of(c, x.own, n_head, type, true);
    x.own_p = split_of(c, x.own, n_head, type, x.own_v, true);
    // One chunk a sequence, which joins the prefix's parts itself, where there are CTAs
    // enough for the length: 16 positions a CTA (behind 1000 positions, f16, 64 heads
    // over 8 of 128, so and in three launches: 4 streams, 32 CTAs, 300 of their own 12.8
    // and 13.6 us, 700 15.8 and 14.6, 1500 21.9 and 14.6; 16 streams, 128 CTAs, 1500
    // 28.5 and 32.4, 2500 38.9 and 42.7, 4000 57.4 and 51.1; 30, 240 CTAs, 2500 51.3
    // and 57.6, 4000 70.9 and 70.3; 4 of f32, 36 heads of 64, 144 CTAs, 1000 15.5 and
    // 19.5, 2500 27.6 and 27.3, 4000 39.6 and 32.0).
    const long long units = (long long)s.n_seq * c.n_kv * x.own_p.row_tiles;
    if (x.pre_p.n_chunk <= MERGE && (x.own.max_len <= 16 * units || units >= 296) && (type == T_F32 || x.own.max_len <= sum_most(type))) {
      x.own_p.n_chunk = 1;
      x.own_p.chunk = (x.own.max_len + 63) / 64 * 64;
      x.merge = true;
    }
  }
  return x;
}
}  // namespace

size_t kv_attn_shared_scratch_bytes(const pk_kv_cache &c, const pk_kv_seqs &seqs, const pk_kv_shared &sh, int n_head, int type) {
  const pk_kv_seqs s = bounded(c, seqs);
  const Shared x = shared_plan(c, s, sh, n_head, type);
  return (size_t)s.n_tok * n_head * (x.pre_p.n_chunk + (x.merge ? 0 : x.own_p.n_chunk)) * (c.head_dim + 2) * sizeof(float);
}

cudaError_t launch_kv_attn_shared(const pk_kv_cache &c, const pk_kv_seqs &seqs, const pk_kv_shared &sh, const pk_kv_query &q,
                                  void *scratch, cudaStream_t st) {
  const pk_kv_seqs s = bounded(c, seqs);
  const Shared x = shared_plan(c, s, sh, q.n_head, q.type);
  const size_t rows = (size_t)s.n_tok * q.n_head;
  if (rows > 0x7fffffff) return cudaErrorInvalidValue;
  AttnKArgs a = args_of(c, s, q);
  a.sh = sh;
  // (The groups stay also where nothing is computed for all of one: what a sequence
  // has besides is counted from its group's shared length, 15 at the most then.)
  a.n_pre = x.pre_p.n_chunk;
  a.pre_chunk = std::max(x.pre_p.chunk, 1);
  a.n_part = a.n_pre + (x.merge ? 0 : x.own_p.n_chunk);
  a.part_o = reinterpret_cast<float *>(scratch);
  a.part_ml = reinterpret_cast<float2 *>(a.part_o + rows * a.n_part * c.head_dim);
  cudaError_t e = cudaSuccess;
  if (a.n_pre > 0) {
    AttnKArgs b = a;
    b.mode = ATTN_PREFIX;
    b.q.mask = nullptr;
    if (x.wide) {
      b.chunk = x.pre_p.chunk; b.n_chunk = x.pre_p.n_chunk; b.row_tiles = x.pre_p.row_tiles;
      const long long blocks = (long long)sh.n_group * c.n_kv * b.row_tiles * b.n_chunk;
      if (blocks > 0x7fffffffLL) return cudaErrorInvalidValue;
      e = launch_kv_prefix(b, (unsigned)blocks, st);
    } else {
      e = launch_parts(b, x.pre_v, x.pre_p, sh.n_group, st);
    }
    if (e != cudaSuccess) return e;
  }
  a.mode = ATTN_OWN;
  a.part0 = a.n_pre;
  a.chunk = 64;
  a.merge = x.merge;
  a.early = a.n_pre > 0;
  if (x.own_p.n_chunk > 0) e = launch_parts(a, x.own_v, x.own_p, s.n_seq, st);
  return e != cudaSuccess || a.merge ? e : launch_join(a, st);
}

}  // namespace pk
