// pk_cache.cu -- the quantised paged K/V cache: rows quantised as they are
// written, read back, and moved when drafts are accepted.  No counterpart in
// the reference, whose cache is f32 (model.rs:352-387).
//
// A row of head_dim values is held by head_dim / 8 lanes, 8 values each, so a
// warp has 2 (head_dim 128) or 4 (64) rows at once: 16-byte loads of half
// precision, 8- or 4-byte stores of codes, each row's bytes contiguous over
// its lanes.  The largest magnitude goes over the row's lanes by shuffles
// (Q4: over the four lanes of each 32 dimensions first).
//
// Measured: 5 prompts of up to 3500 tokens, 36 heads of 64, f16 into Q4 and
// back, 59 us for both (memory alone: 33); 10800 rows of 36 heads of 64 alone:
// f16 into Q4 51 us and back 33 (20 each), f32 into Q8 64 and back 66 (39); 64
// rows of 8 heads of 128 are the launches.  What bounds the store is the codes' exact rounding.
#include "pk_cache.cuh"
#include "pk_cache.h"
#include "pk_launch.h"

namespace pk {
namespace {

constexpr int CT = 128;  // threads of a CTA

// (a0 b0 + c0, a1 b1 + c1), rounded once each, in one instruction.
__device__ __forceinline__ void fma_x2(float a0, float a1, float b0, float b1, float c0, float c1, float &d0, float &d1) {
  asm("{\n .reg .b64 a, b, c;\n mov.b64 a, {%2, %3};\n mov.b64 b, {%4, %5};\n mov.b64 c, {%6, %7};\n"
      " fma.rn.f32x2 a, a, b, c;\n mov.b64 {%0, %1}, a;\n}"
      : "=f"(d0), "=f"(d1)
      : "f"(a0), "f"(a1), "f"(b0), "f"(b1), "f"(c0), "f"(c1));
}

// The codes of a lane's eight values, round(x / d) to even, as the bits of
// 1.5 2^23 + c (whose last bits are c's); most: the largest code.  The product
// with an approximate reciprocal lies within 2^-15 of the quotient (below 128;
// the reciprocal's error and the rounding), so c is off by at most one, and
// only where x lies within 2^-14 of a step of the middle between two codes.
// There the remainder x - d c, exact in f32 (both terms are multiples of the
// smaller one's last place and the difference is below 2 d), tells on which
// side.  Scales near f32's lower end are moved up with their values first;
// below its normal range D itself is coarse and quotients may pass `most`.
__device__ __forceinline__ void codes8(float (&x)[8], float d, float most, uint32_t (&u)[8]) {
  const bool tiny = !(d >= 0x1p-60f);
  if (tiny) {
#pragma unroll
    for (int i = 0; i < 8; i++) x[i] = d > 0.0f ? x[i] * 0x1p64f : 0.0f;
    d = d > 0.0f ? d * 0x1p64f : 1.0f;
  }
  float inv, far = 0.0f;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(inv) : "f"(d));
#pragma unroll
  for (int i = 0; i < 8; i += 2) {
    float t0, t1, c0, c1, r0, r1;
    fma_x2(x[i], x[i + 1], inv, inv, 12582912.0f, 12582912.0f, t0, t1);
    fma_x2(t0, t1, -1.0f, -1.0f, 12582912.0f, 12582912.0f, c0, c1);  // -c
    fma_x2(c0, c1, d, d, x[i], x[i + 1], r0, r1);
    u[i] = __float_as_uint(t0);
    u[i + 1] = __float_as_uint(t1);
    far = fmaxf(far, fmaxf(fabsf(r0), fabsf(r1)));
  }
  if (tiny || far >= d * (0.5f - 0x1p-14f)) {
#pragma unroll
    for (int i = 0; i < 8; i++) {
      float c = fsub(__uint_as_float(u[i]), 12582912.0f);
      const float r = __fmaf_rn(-d, c, x[i]), h = 0.5f * d, a = fabsf(r);
      if (a > h || (a == h && (u[i] & 1u))) c += r > 0.0f ? 1.0f : -1.0f;
      c = fminf(fmaxf(c, most < 127.0f ? -8.0f : -127.0f), most);
      u[i] = __float_as_uint(fadd(c, 12582912.0f));
    }
  }
}
// m / c for c = 127, 105 as the division rounds it (Markstein: one correction
// of the product with the rounded reciprocal by the exact remainder; equal to
// the division for every 24-bit significand), or by it near the ends.
__device__ __forceinline__ float over(float m, float c, float rc) {
  if (!(m >= 0x1p-90f)) return fdiv(m, c);
  const float q = fmul(m, rc);
  return __fmaf_rn(__fmaf_rn(-c, q, m), rc, q);
}

struct RowsArgs {
  pk_kv_cache c;
  pk_kv_seqs s;
  const void *src[2];
  void *dst[2];
  long tok_stride, head_stride;
  int vec, parts, sets;  // parts: warps a token; sets: row sets a warp (a multiple of U)
};

// A warp has one token and some sets of RW heads, K and V of each, U sets at a
// time: the rows' values are asked for before the token's sequence, position
// and page are looked up, a chain of four dependent reads that is the same for
// all of them, and from set to set only additions lead.
constexpr int U = 2;
struct Place {
  int t, set0, lane, l;
};
__device__ __forceinline__ Place place_of(const RowsArgs &a, int L) {
  const long long w = (long long)blockIdx.x * (CT / 32) + (threadIdx.x >> 5);
  Place p;
  p.t = (int)(w / a.parts);
  p.set0 = (int)(w - (long long)p.t * a.parts) * a.sets;
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

// Quantises a row held eight values a lane and writes it: codes at `codes`
// (this lane's), scale at `scale` (the row's).  All lanes of the warp call it.
template <int TYPE, int DH, class E>
__device__ __forceinline__ void store_row(const uint4 (&raw)[sizeof(E) / 2], bool on, int lane, int l, uint8_t *codes, float *scale) {
  constexpr int L = DH / 8;
  float x[8];
  uint32_t mb = 0;  // bits of the largest magnitude: NaN's are above infinity's
#pragma unroll
  for (int i = 0; i < 8; i++) x[i] = to_f(reinterpret_cast<const E *>(raw)[i]);
  if (sizeof(E) == 2) {  // two at a time
    const uint32_t m2 = __vmaxu2(__vmaxu2(raw[0].x & 0x7fff7fffu, raw[0].y & 0x7fff7fffu),
                                 __vmaxu2(raw[0].z & 0x7fff7fffu, raw[0].w & 0x7fff7fffu));
    const uint16_t m1 = (uint16_t)max(m2 >> 16, m2 & 0xffffu);
    mb = __float_as_uint(to_f(*reinterpret_cast<const E *>(&m1))) & 0x7fffffffu;
  } else {
#pragma unroll
    for (int i = 0; i < 8; i++) mb = max(mb, __float_as_uint(x[i]) & 0x7fffffffu);
  }
  if (mb > 0x7f000000u) {  // 2^127
    mb = 0;
#pragma unroll
    for (int i = 0; i < 8; i++) {
      x[i] = isnan(x[i]) ? 0.0f : fminf(fmaxf(x[i], -0x1p127f), 0x1p127f);
      mb = max(mb, __float_as_uint(x[i]) & 0x7fffffffu);
    }
  }
  uint32_t u[8];
  if (TYPE == PK_KV_Q8) {
#pragma unroll
    for (int o = L / 2; o > 0; o >>= 1) mb = max(mb, __shfl_xor_sync(0xffffffffu, mb, o));
    const float d = over(__uint_as_float(mb), 127.0f, 1.0f / 127.0f);
    codes8(x, d, 127.0f, u);
    uint32_t w[2];
#pragma unroll
    for (int i = 0; i < 2; i++)
      w[i] = __byte_perm(__byte_perm(u[4 * i], u[4 * i + 1], 0x0040), __byte_perm(u[4 * i + 2], u[4 * i + 3], 0x0040), 0x5410) ^ 0x80808080u;
    if (on) {
      *reinterpret_cast<uint2 *>(codes) = make_uint2(w[0], w[1]);
      if (l == 0) *scale = d;
    }
  } else {
#pragma unroll
    for (int o = 2; o > 0; o >>= 1) mb = max(mb, __shfl_xor_sync(0xffffffffu, mb, o));
    const float block = __uint_as_float(mb);  // of the 32 dimensions
#pragma unroll
    for (int o = L / 2; o > 2; o >>= 1) mb = max(mb, __shfl_xor_sync(0xffffffffu, mb, o));
    const float d = over(__uint_as_float(mb), 105.0f, 1.0f / 105.0f);
    // ceil of the rounded quotient block / (7 d), 1 .. 15 (1 for d = 0): the
    // division itself only where a quotient 2^-20 off could change it
    const float d7 = fmul(7.0f, d);
    float inv, sb = 15.0f;
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(inv) : "f"(d7));
    const float q = fmul(block, inv), near = rintf(q);
    if (!(d >= 0x1p-100f) || (fabsf(q - near) < 0x1p-16f && near < 15.0f))
      sb = d > 0.0f ? fminf(fmaxf(ceilf(fdiv(block, d7)), 1.0f), 15.0f) : 1.0f;
    else if (q < 14.5f)
      sb = fmaxf(ceilf(q), 1.0f);
    codes8(x, fmul(d, sb), 7.0f, u);
    uint32_t w = 0x88888888u - 0x4b400000u * 0x11111111u;  // sum of (c + 8) 16^i, by the words' last bits
#pragma unroll
    for (int i = 0; i < 8; i++) w += u[i] << (4 * i);
    uint32_t word = (uint32_t)sb << (4 * (l / 4));
    word |= __shfl_xor_sync(0xffffffffu, word, 4);
    if (DH == 128) word |= __shfl_xor_sync(0xffffffffu, word, 8);
    if (on) {
      *reinterpret_cast<uint32_t *>(codes) = w;
      if (l == 0) *reinterpret_cast<float2 *>(scale) = make_float2(d, __uint_as_float(word));
    }
  }
}

template <int TYPE, int DH, int T>
__global__ void __launch_bounds__(CT, 8) k_kv_store(const RowsArgs a) {
  using E = elem_t<T>;
  constexpr int L = DH / 8, RW = 32 / L, RB = TYPE == PK_KV_Q8 ? DH : DH / 2, SW = TYPE == PK_KV_Q8 ? 1 : 2, W = sizeof(E) / 2;
  pdl_trigger();
  pdl_wait();
  const Place pl = place_of(a, L);
  if (pl.t >= a.s.n_tok) return;
  const int set1 = min(pl.set0 + a.sets, (a.c.n_kv + RW - 1) / RW);
  int h = pl.set0 * RW + pl.lane / L;
  const long long off = (long long)pl.t * a.tok_stride + (long long)h * a.head_stride + 8 * pl.l, step = RW * a.head_stride;
  const E *k = reinterpret_cast<const E *>(a.src[0]) + off, *v = reinterpret_cast<const E *>(a.src[1]) + off;
  uint4 rk[U][W], rv[U][W];
  auto ask1 = [&](uint4(&raw)[W], const E *p) {
    if (a.vec) {
#pragma unroll
      for (int w = 0; w < W; w++) raw[w] = __ldg(reinterpret_cast<const uint4 *>(p) + w);
    } else {
#pragma unroll
      for (int i = 0; i < 8; i++) reinterpret_cast<E *>(raw)[i] = p[i];
    }
  };
  auto ask = [&](int h) {  // the next U sets
#pragma unroll
    for (int i = 0; i < U; i++) {
#pragma unroll
      for (int w = 0; w < W; w++) rk[i][w] = rv[i][w] = make_uint4(0, 0, 0, 0);
      if (h + i * RW >= a.c.n_kv) continue;
      ask1(rk[i], k);
      ask1(rv[i], v);
      k += step;
      v += step;
    }
  };
  ask(h);
  bool mine;
  const long long row0 = head0_row(a, pl.t, pl.lane, &mine);
  if (row0 < 0) return;
  const size_t row = (size_t)row0 + (size_t)h * a.c.page_size, rows = (size_t)RW * a.c.page_size;
  size_t co = row * RB + pl.l * (RB / L), so = row * SW;
  for (int set = pl.set0; set < set1; set += U) {
    if (set > pl.set0) ask(h);
#pragma unroll
    for (int i = 0; i < U; i++) {
      if (set + i >= set1) break;  // (the whole warp)
      const bool on = h < a.c.n_kv;
      store_row<TYPE, DH, E>(rk[i], on, pl.lane, pl.l, reinterpret_cast<uint8_t *>(a.c.k) + co, a.c.ks + so);
      store_row<TYPE, DH, E>(rv[i], on, pl.lane, pl.l, reinterpret_cast<uint8_t *>(a.c.v) + co, a.c.vs + so);
      co += rows * RB;
      so += rows * SW;
      h += RW;
    }
  }
}

template <int TYPE, int DH, int T>
__global__ void __launch_bounds__(CT) k_kv_load(const RowsArgs a) {
  using E = elem_t<T>;
  constexpr int L = DH / 8, RW = 32 / L, RB = TYPE == PK_KV_Q8 ? DH : DH / 2, SW = TYPE == PK_KV_Q8 ? 1 : 2;
  pdl_trigger();
  pdl_wait();
  const Place pl = place_of(a, L);
  if (pl.t >= a.s.n_tok) return;
  bool mine;
  const long long row0 = head0_row(a, pl.t, pl.lane, &mine);
  if (!mine) return;
  const int h0 = pl.set0 * RW + pl.lane / L, h1 = min(a.c.n_kv, (pl.set0 + a.sets) * RW);
  const size_t row = (size_t)max(row0, 0LL) + (size_t)h0 * a.c.page_size, rows = (size_t)RW * a.c.page_size;
  size_t co = row * RB + pl.l * (RB / L), so = row * SW;
  long long off = (long long)pl.t * a.tok_stride + (long long)h0 * a.head_stride + 8 * pl.l;
  for (int h = h0; h < h1; h += U * RW) {
    uint2 u[U][2];
    float2 d[U][2];
#pragma unroll
    for (int i = 0; i < U; i++) {
#pragma unroll
      for (int w = 0; w < 2; w++) {
        u[i][w] = make_uint2(0x80808080u, 0x80808080u);
        d[i][w] = make_float2(0.0f, 0.0f);  // no page: D = 0
        if (row0 < 0 || h + i * RW >= h1) continue;
        const uint8_t *codes = reinterpret_cast<const uint8_t *>(w ? a.c.v : a.c.k) + co;
        const float *scales = (w ? a.c.vs : a.c.ks) + so;
        if (TYPE == PK_KV_Q8) {
          u[i][w] = *reinterpret_cast<const uint2 *>(codes);
          d[i][w].x = *scales;
        } else {
          u[i][w].x = *reinterpret_cast<const uint32_t *>(codes);
          d[i][w] = *reinterpret_cast<const float2 *>(scales);
        }
      }
      co += rows * RB;
      so += rows * SW;
    }
#pragma unroll
    for (int i = 0; i < U; i++) {
      if (h + i * RW >= h1) break;
#pragma unroll
      for (int w = 0; w < 2; w++) {
        float x[8];
        const float dd = d[i][w].x;
        if (TYPE == PK_KV_Q8) {
#pragma unroll
          for (int e = 0; e < 4; e++) {
            const float2 f = __half22float2(u2h(codes_of(e < 2 ? u[i][w].x : u[i][w].y, e % 2 ? 0x4342 : 0x4140)));
            x[2 * e] = fmul(dd, f.x);
            x[2 * e + 1] = fmul(dd, f.y);
          }
        } else {
          const int sb = (int)((__float_as_uint(d[i][w].y) >> (4 * (pl.l / 4))) & 15u);
          const uint32_t s2 = dup_h(sb), m2 = dup_h(-1032 * sb);
#pragma unroll
          for (int e = 0; e < 4; e++) {  // nibbles e and e + 4
            const float2 f = __half22float2(u2h(nibbles_of(u[i][w].x >> (4 * e), s2, m2)));
            x[e] = fmul(dd, f.x);
            x[e + 4] = fmul(dd, f.y);
          }
        }
        store_n<E, 8>(reinterpret_cast<E *>(a.dst[w]) + off, a.vec, x);
      }
      off += RW * a.head_stride;
    }
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
  // U sets a warp, or all where that still gives every SM 48 warps: the
  // look-ups are then shared by more rows
  const int all = (a.c.n_kv + rw - 1) / rw;
  a.sets = U;
  while (a.sets < all && (long long)a.s.n_tok * ((all + 2 * a.sets - 1) / (2 * a.sets)) >= 148 * 48) a.sets *= 2;
  a.parts = (all + a.sets - 1) / a.sets;
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
