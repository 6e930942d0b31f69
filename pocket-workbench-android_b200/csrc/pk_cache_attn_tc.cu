// pk_cache_attn_tc.cu -- attention over the quantised cache for many query
// rows of a kv head (drafted trees, prompt chunks; half-precision queries) on
// the fifth-generation tensor cores.  The formulas are pk_cache_attn.cu's.
//
// A CTA takes 128 rows (token, query head) of one kv head over one chunk of
// positions, 64 at a time: S = Q K^T (M 128 x N 64 x K head_dim) into one of
// two TMEM buffers, weights P, O += P V (M 128 x N head_dim x K 64) in TMEM.
// 256 threads:
//   warps 0-3  softmax: thread = row = TMEM lane.  Scores from TMEM, the
//              scales D^K and D^V applied in f32 (two at a time), weights as
//              f16 into shared memory.  O stays in TMEM; a row's is scaled
//              there only when its factor has to change (M grew past 2^100,
//              or weights would leave f16), which is rare after the first
//              tiles, and M itself moves by 2^6 at least.
//   warps 4-7  codes: the next tiles' K and V rows on their way in registers,
//              made f16 (exact) and put into the operands' layout; warp 4
//              issues the products.
// Two CTAs share an SM (96 KB and 256 TMEM columns each), so that one's
// products run beside the other's softmax.  Operands are in the canonical
// layout without swizzle, core matrices of 8 rows x 16 bytes: 16-byte chunks of
// consecutive rows are consecutive, and a warp's stores (a lane a row) touch
// every bank once.  V's rows are stored as K's, which makes it an N-major
// operand.
//
// Every wait is bounded: one that runs out sets the CTA's abort flag, after
// which no wait waits, and its rows are written as NaN.
#include <algorithm>

#include "pk_cache_attn.cuh"
#include "pk_tcgen05.cuh"

namespace pk {
namespace {

constexpr int NK = 64;                      // positions a tile
constexpr int ROWS = TC_ATTN_ROWS;
constexpr int SOFT = 128, CONV = 128;       // threads
constexpr unsigned long long WAIT_NS = 2000000000ull;

template <int DH>
struct Lay {
  static constexpr int Q = 0, K = Q + ROWS * DH * 2, V = K + 2 * NK * DH * 2, P = V + NK * DH * 2, SC = P + ROWS * NK * 2;
  // of two tiles: D^K [NK], D^V [NK]; positions that hold something (2 words), largest and smallest D^V of 32 (2 x 2)
  static constexpr int SCB = 2 * NK * 4 + 16 + 16, BAR = SC + 2 * SCB, BYTES = BAR + 64;
  static constexpr int S_COL = 0, O_COL = 2 * NK, COLS = 256;
};

__device__ __forceinline__ bool wait(uint32_t bar, uint32_t parity, volatile int *abort) {
  if (mbar_test(bar, parity)) return true;
  const unsigned long long t0 = gtime_ns();
  while (!mbar_test(bar, parity)) {
    if (*abort) return false;
    if (gtime_ns() - t0 > WAIT_NS) {
      *abort = 1;
      return false;
    }
  }
  return true;
}

// A descriptor of an operand without swizzle (pk_tcgen05.cuh): K-major a =
// bytes between the 16-byte halves of a step's K, b = between groups of 8
// rows; N-major a = between groups of 8 k, b = between groups of 8 n.
template <int N, bool BMN>
__device__ __forceinline__ void mma_f16(uint32_t d, uint64_t a, uint64_t b, bool acc) {
  // f32 sums, f16 operands, B N-major when BMN, M 128
  constexpr uint32_t idesc = (1u << 4) | ((BMN ? 1u : 0u) << 16) | ((uint32_t)(N >> 3) << 17) | ((uint32_t)(128 >> 4) << 24);
  asm volatile(
      "{\n .reg .pred p, e;\n elect.sync _|e, 0xffffffff;\n setp.ne.b32 p, %4, 0;\n"
      " @e tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, {%5, %6, %7, %8}, p;\n}" ::"r"(d),
      "l"(a), "l"(b), "r"(idesc), "r"((uint32_t)acc), "r"(0), "r"(0), "r"(0), "r"(0)
      : "memory");
}
// 32 consecutive TMEM columns of this thread's lane.
__device__ __forceinline__ void ld32(uint32_t t, float (&v)[32]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,%20,%21,"
      "%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];\n tcgen05.wait::ld.sync.aligned;"
      : "=f"(v[0]), "=f"(v[1]), "=f"(v[2]), "=f"(v[3]), "=f"(v[4]), "=f"(v[5]), "=f"(v[6]), "=f"(v[7]), "=f"(v[8]), "=f"(v[9]),
        "=f"(v[10]), "=f"(v[11]), "=f"(v[12]), "=f"(v[13]), "=f"(v[14]), "=f"(v[15]), "=f"(v[16]), "=f"(v[17]), "=f"(v[18]),
        "=f"(v[19]), "=f"(v[20]), "=f"(v[21]), "=f"(v[22]), "=f"(v[23]), "=f"(v[24]), "=f"(v[25]), "=f"(v[26]), "=f"(v[27]),
        "=f"(v[28]), "=f"(v[29]), "=f"(v[30]), "=f"(v[31])
      : "r"(t)
      : "memory");
}
__device__ __forceinline__ void st32(uint32_t t, const float (&v)[32]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,%20,%21,"
      "%22,%23,%24,%25,%26,%27,%28,%29,%30,%31,%32};\n tcgen05.wait::st.sync.aligned;" ::"r"(t),
      "f"(v[0]), "f"(v[1]), "f"(v[2]), "f"(v[3]), "f"(v[4]), "f"(v[5]), "f"(v[6]), "f"(v[7]), "f"(v[8]), "f"(v[9]), "f"(v[10]),
      "f"(v[11]), "f"(v[12]), "f"(v[13]), "f"(v[14]), "f"(v[15]), "f"(v[16]), "f"(v[17]), "f"(v[18]), "f"(v[19]), "f"(v[20]),
      "f"(v[21]), "f"(v[22]), "f"(v[23]), "f"(v[24]), "f"(v[25]), "f"(v[26]), "f"(v[27]), "f"(v[28]), "f"(v[29]), "f"(v[30]),
      "f"(v[31])
      : "memory");
}
__device__ __forceinline__ float2 mul2(float2 a, float2 b) {
  float2 d;
  asm("{\n .reg .b64 a, b;\n mov.b64 a, {%2, %3};\n mov.b64 b, {%4, %5};\n mul.rn.f32x2 a, a, b;\n mov.b64 {%0, %1}, a;\n}"
      : "=f"(d.x), "=f"(d.y)
      : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
  return d;
}
__device__ __forceinline__ float2 add2(float2 a, float2 b) {
  float2 d;
  asm("{\n .reg .b64 a, b;\n mov.b64 a, {%2, %3};\n mov.b64 b, {%4, %5};\n add.rn.f32x2 a, a, b;\n mov.b64 {%0, %1}, a;\n}"
      : "=f"(d.x), "=f"(d.y)
      : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
  return d;
}
__device__ __forceinline__ float2 fma2(float2 a, float2 b, float2 c) {
  float2 d;
  asm("{\n .reg .b64 a, b, c;\n mov.b64 a, {%2, %3};\n mov.b64 b, {%4, %5};\n mov.b64 c, {%6, %7};\n"
      " fma.rn.f32x2 a, a, b, c;\n mov.b64 {%0, %1}, a;\n}"
      : "=f"(d.x), "=f"(d.y)
      : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y), "f"(c.x), "f"(c.y));
  return d;
}

// The order of a word's eight dimensions in an operand: as they lie for Q8, as
// the nibble pairs (i, i + 4) come out for Q4.
template <int TYPE>
__host__ __device__ constexpr int dim8(int i) {
  return TYPE == PK_KV_Q8 ? i : (i / 2) + 4 * (i % 2);
}

// 16 bytes of a row's codes into 16-byte chunks of f16 at dst, `stride` apart.
template <int TYPE>
__device__ __forceinline__ void put_codes(uint32_t dst, uint32_t stride, const uint4 &raw, uint32_t s2, uint32_t m2) {
  const uint32_t w[4] = {raw.x, raw.y, raw.z, raw.w};
  if (TYPE == PK_KV_Q8) {
#pragma unroll
    for (int c = 0; c < 2; c++)
      sts128(dst + c * stride, codes_of(w[2 * c], 0x4140), codes_of(w[2 * c], 0x4342), codes_of(w[2 * c + 1], 0x4140),
             codes_of(w[2 * c + 1], 0x4342));
  } else {
#pragma unroll
    for (int c = 0; c < 4; c++)
      sts128(dst + c * stride, nibbles_of(w[c], s2, m2), nibbles_of(w[c] >> 4, s2, m2), nibbles_of(w[c] >> 8, s2, m2),
             nibbles_of(w[c] >> 12, s2, m2));
  }
}

// This thread's query row, scaled to |q'| < 2 and rounded to f16 (exact for
// f16 and bf16 down to 2^-24 of the row's largest), into the operand; its r.
template <int TYPE, int DH, class E>
__device__ __forceinline__ float put_q(const AttnKArgs &a, const Unit &u, int row, uint32_t dst) {
  const bool on = row < u.rows;
  const int i = row / a.group, h = u.h * a.group + row - i * a.group;
  const E *p = reinterpret_cast<const E *>(a.q.q) + (on ? (long long)(u.sv.first + i) * a.q.q_tok_stride + (long long)h * a.q.q_head_stride : 0);
  float m = 0.0f;
  if (on) {
#pragma unroll
    for (int c = 0; c < DH / 8; c++) {
      float x[8];
      load_n<E, 8>(p + 8 * c, a.vec_q, x);
#pragma unroll
      for (int j = 0; j < 8; j++) m = fmaxf(m, fabsf(x[j]));
    }
  }
  int e = (int)(__float_as_uint(m) >> 23) - 127;
  e = m > 0.0f ? min(max(e, -100), 126) : 0;
  const float up = __int_as_float((e + 127) << 23), down = __int_as_float((127 - e) << 23);
#pragma unroll
  for (int c = 0; c < DH / 8; c++) {
    uint32_t w[4] = {0, 0, 0, 0};
    if (on) {
      float x[8];
      load_n<E, 8>(p + 8 * c, a.vec_q, x);
#pragma unroll
      for (int j = 0; j < 4; j++) w[j] = pack2(x[dim8<TYPE>(2 * j)] * down, x[dim8<TYPE>(2 * j + 1)] * down);
    }
    sts128(dst + c * (ROWS * 16), w[0], w[1], w[2], w[3]);
  }
  return a.q.scale * kLog2e * up;
}

// Which of positions p0 .. p0 + 63 token i sees (bit by position).
__device__ __forceinline__ uint64_t seen_by(const AttnKArgs &a, const Unit &u, int i, int p0, int hi) {
  auto ones = [](int n) { return n >= 64 ? ~0ull : n <= 0 ? 0ull : (1ull << n) - 1; };
  uint64_t v = ones(u.sv.ctx - p0);
  const int j0 = p0 - u.sv.ctx;  // draft at p0
  if (!a.q.mask) {
    v = ones(u.sv.ctx + i + 1 - p0);
  } else if (j0 + 63 >= 0) {
    const uint64_t *w = a.q.mask + (size_t)(u.sv.first + i) * a.q.mask_words;
    uint64_t d;
    if (j0 < 0) {
      d = __ldg(w) << (-j0);
    } else {
      const int k = j0 >> 6, sh = j0 & 63;
      d = k < a.q.mask_words ? __ldg(w + k) >> sh : 0;
      if (sh && k + 1 < a.q.mask_words) d |= __ldg(w + k + 1) << (64 - sh);
    }
    v |= d;
  }
  return v & ones(hi - p0) & ones(u.sv.ctx + u.sv.n - p0);
}

template <int TYPE, int DH>
__global__ void __launch_bounds__(SOFT + CONV, 2) k_kv_attn_tc(const AttnKArgs a) {
  using L = Lay<DH>;
  constexpr int RB = TYPE == PK_KV_Q8 ? DH : DH / 2, SW = TYPE == PK_KV_Q8 ? 1 : 2;
  constexpr int W = RB / 32;  // 16-byte words of half a row
  extern __shared__ __align__(1024) uint8_t smem[];
  pdl_wait();
  const Unit u = unit_of(a);
  const int tile0 = u.rt * ROWS;
  if (u.ch >= max(u.nch, 1) || tile0 >= u.rows) {
    pdl_trigger();
    return;
  }
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const uint32_t sb = shaddr(smem);
  // barriers: S full x 2, scales ready x 2, P ready, PV done; the TMEM address; the abort flag
  const uint32_t bar = sb + L::BAR, sfull = bar, scready = bar + 16, pready = bar + 32, pvdone = bar + 40;
  volatile int *abort = reinterpret_cast<volatile int *>(smem + L::BAR + 52);
  if (tid == 0) {
    mbar_init(sfull, 1);
    mbar_init(sfull + 8, 1);
    mbar_init(scready, CONV);
    mbar_init(scready + 8, CONV);
    mbar_init(pready, SOFT);
    mbar_init(pvdone, 1);
    *abort = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (warp == 4) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(bar + 48), "r"(L::COLS) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  const int row = tile0 + tid;
  float rs = 0.0f;
  if (tid < SOFT) {
    const uint32_t dst = sb + L::Q + tid * 16;
    rs = a.q.type == T_F16 ? put_q<TYPE, DH, __half>(a, u, row, dst) : put_q<TYPE, DH, __nv_bfloat16>(a, u, row, dst);
    fence_async_smem();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  pdl_trigger();
  const uint32_t tmem = *reinterpret_cast<volatile uint32_t *>(smem + L::BAR + 48);
  // without a mask nobody sees past the tile's last token
  const int last = (min(tile0 + ROWS, u.rows) - 1) / a.group;
  const int hi = a.q.mask ? u.hi : min(u.hi, u.sv.ctx + last + 1);
  const int nt = hi > u.lo ? (hi - u.lo + NK - 1) / NK : 0;

  if (tid >= SOFT) {  // -------------------------------------------------- codes
    const int ct = tid - SOFT, key = ct & (NK - 1), half = ct >> 6;
    uint4 rk[W], rv[W];
    float2 dk, dv;  // (D, sub-scales)
    bool on = false;
    auto page_of = [&](int i) {
      const int p = u.lo + NK * i + key, j = p >> a.page_shift;
      const int pg = i < nt && p < hi && j < a.s.max_pages ? __ldg(a.s.pages + (size_t)u.s * a.s.max_pages + j) : -1;
      return pg >= 0 && pg < a.c.n_pages ? pg : -1;
    };
    auto row_of = [&](int i, int pg) {
      const int p = u.lo + NK * i + key;
      return ((size_t)pg * a.c.n_kv + u.h) * a.c.page_size + (p & (a.c.page_size - 1));
    };
    auto ask = [&](uint4(&raw)[W], float2 &d, const void *codes, const float *scales, int i, int pg) {
#pragma unroll
      for (int w = 0; w < W; w++) raw[w] = TYPE == PK_KV_Q8 ? make_uint4(0x80808080u, 0x80808080u, 0x80808080u, 0x80808080u)
                                                           : make_uint4(0x88888888u, 0x88888888u, 0x88888888u, 0x88888888u);
      d = make_float2(0.0f, 0.0f);
      if (pg < 0) return;
      const size_t r = row_of(i, pg);
      const uint4 *src = reinterpret_cast<const uint4 *>(reinterpret_cast<const uint8_t *>(codes) + r * RB) + half * W;
#pragma unroll
      for (int w = 0; w < W; w++) raw[w] = __ldg(src + w);
      if (TYPE == PK_KV_Q8) d.x = __ldg(scales + r);
      else d = __ldg(reinterpret_cast<const float2 *>(scales) + r);
    };
    auto put = [&](uint32_t dst, const uint4(&raw)[W], float2 d) {
#pragma unroll
      for (int w = 0; w < W; w++) {
        constexpr int CW = TYPE == PK_KV_Q8 ? 2 : 4;  // chunks of 16 bytes of codes
        const int chunk = (half * W + w) * CW;
        uint32_t s2 = 0, m2 = 0;
        if (TYPE == PK_KV_Q4) {  // 16 bytes are 32 dimensions: one sub-scale
          const int s = (int)((__float_as_uint(d.y) >> (4 * (half * W + w))) & 15u);
          s2 = dup_h(s);
          m2 = dup_h(-1032 * s);
        }
        put_codes<TYPE>(dst + chunk * (NK * 16) + key * 16, NK * 16, raw[w], s2, m2);
      }
    };
    // K's codes and both scales of tile i, and the tile's summary
    auto put_k = [&](int i) {
      const int b = i & 1;
      put(sb + L::K + b * (NK * DH * 2), rk, dk);
      uint8_t *sc = smem + L::SC + b * L::SCB;
      if (half == 0) {
        reinterpret_cast<float *>(sc)[key] = dk.x;
        const unsigned m = __ballot_sync(0xffffffffu, on);
        if (lane == 0) reinterpret_cast<uint32_t *>(sc + 2 * NK * 4)[key >> 5] = m;
      } else {
        reinterpret_cast<float *>(sc)[NK + key] = dv.x;
        const uint32_t hi_v = __reduce_max_sync(0xffffffffu, __float_as_uint(dv.x) & 0x7fffffffu);
        const uint32_t lo_v = __reduce_min_sync(0xffffffffu, dv.x > 0.0f ? __float_as_uint(dv.x) : 0x7f800000u);
        if (lane == 0) {
          reinterpret_cast<uint32_t *>(sc + 2 * NK * 4 + 16)[key >> 5] = hi_v;
          reinterpret_cast<uint32_t *>(sc + 2 * NK * 4 + 24)[key >> 5] = lo_v;
        }
      }
      mbar_arrive(scready + 8 * b);
    };
    int pg = page_of(0), next = page_of(1);
    ask(rk, dk, a.c.k, a.c.ks, 0, pg);
    ask(rv, dv, a.c.v, a.c.vs, 0, pg);
    on = pg >= 0;
    if (nt > 0) {
      put_k(0);
      put(sb + L::V, rv, dv);
      // from here rk, dk hold tile i + 1's K during iteration i, rv, dv its V
      pg = next;
      next = page_of(2);
      ask(rk, dk, a.c.k, a.c.ks, 1, pg);
      ask(rv, dv, a.c.v, a.c.vs, 1, pg);
      on = pg >= 0;
    }
    auto scores = [&](int i) {  // warp 4
      const uint32_t k = sb + L::K + (i & 1) * (NK * DH * 2), d = tmem + L::S_COL + (i & 1) * NK;
#pragma unroll
      for (int s = 0; s < DH / 16; s++)
        mma_f16<NK, false>(d, tc_desc(sb + L::Q + s * 2 * (ROWS * 16), ROWS * 16, 128), tc_desc(k + s * 2 * (NK * 16), NK * 16, 128), s > 0);
      tc_commit(sfull + 8 * (i & 1));
    };
    if (nt > 0) {
      fence_async_smem();
      asm volatile("bar.sync 1, %0;" ::"n"(CONV) : "memory");
      if (warp == 4) {
        tc_fence_after();
        scores(0);
      }
    }
    for (int i = 0; i < nt; i++) {
      if (i + 1 < nt) put_k(i + 1);
      fence_async_smem();
      asm volatile("bar.sync 1, %0;" ::"n"(CONV) : "memory");
      if (warp == 4) {
        if (i + 1 < nt) scores(i + 1);
        wait(pready, i & 1, abort);
        tc_fence_after();
#pragma unroll
        for (int s = 0; s < NK / 16; s++)
          mma_f16<DH, true>(tmem + L::O_COL, tc_desc(sb + L::P + s * 2 * (ROWS * 16), ROWS * 16, 128),
                            tc_desc(sb + L::V + s * 16 * 16, 128, NK * 16), i > 0 || s > 0);
        tc_commit(pvdone);
      }
      if (i + 1 < nt) {
        // tile i + 2's K may be asked for; V's registers are free once tile i + 1's is stored
        const int pg2 = next;
        next = page_of(i + 3);
        ask(rk, dk, a.c.k, a.c.ks, i + 2, pg2);
        wait(pvdone, i & 1, abort);
        put(sb + L::V, rv, dv);
        ask(rv, dv, a.c.v, a.c.vs, i + 2, pg2);
        on = pg2 >= 0;
      }
    }
  } else {  // ------------------------------------------------------------ softmax
    const uint32_t lanes = (uint32_t)(warp * 32) << 16;
    const bool work = tile0 + warp * 32 < u.rows;  // (the whole warp)
    const int tok = min(row, u.rows - 1) / a.group;
    float m = -CUDART_INF_F, l = 0.0f, inv = 0x1p100f;
    // O's row times f, once the products before are done (i > 0)
    auto scale_o = [&](int i, float f) {
      if (i == 0) return;
      wait(pvdone, (i - 1) & 1, abort);
      tc_fence_after();
#pragma unroll
      for (int c = 0; c < DH / 32; c++) {
        float v[32];
        ld32(tmem + lanes + L::O_COL + 32 * c, v);
#pragma unroll
        for (int j = 0; j < 32; j++) v[j] *= f;
        st32(tmem + lanes + L::O_COL + 32 * c, v);
      }
    };
    for (int i = 0; i < nt; i++) {
      const int b = i & 1, p0 = u.lo + NK * i;
      wait(scready + 8 * b, (i >> 1) & 1, abort);
      wait(sfull + 8 * b, (i >> 1) & 1, abort);
      tc_fence_after();
      if (work) {
        const uint8_t *sc = smem + L::SC + b * L::SCB;
        const float4 *dk4 = reinterpret_cast<const float4 *>(sc), *dv4 = reinterpret_cast<const float4 *>(sc + NK * 4);
        const uint64_t held = *reinterpret_cast<const uint64_t *>(sc + 2 * NK * 4);
        const uint4 r4 = *reinterpret_cast<const uint4 *>(sc + 2 * NK * 4 + 16);
        const float vmax = fmaxf(__uint_as_float(r4.x), __uint_as_float(r4.y)), vmin = fminf(__uint_as_float(r4.z), __uint_as_float(r4.w));
        const bool masked = p0 + NK > min(u.sv.ctx, hi) || held != ~0ull;
        // per weight where scales differ so much that the largest says little about the others
        const bool each = masked || !(vmax <= 65536.0f * vmin);
        float t[NK];
        ld32(tmem + lanes + L::S_COL + NK * b, reinterpret_cast<float(&)[32]>(t[0]));
        ld32(tmem + lanes + L::S_COL + NK * b + 32, reinterpret_cast<float(&)[32]>(t[32]));
        float2 *t2 = reinterpret_cast<float2 *>(t);
#pragma unroll
        for (int j = 0; j < NK / 4; j++) {
          const float4 d = dk4[j];
          t2[2 * j] = mul2(t2[2 * j], make_float2(d.x, d.y));
          t2[2 * j + 1] = mul2(t2[2 * j + 1], make_float2(d.z, d.w));
        }
        uint64_t vis = ~0ull;
        if (masked) {
          vis = held & (row < u.rows ? seen_by(a, u, tok, p0, hi) : 0);
#pragma unroll
          for (int j = 0; j < NK; j++)
            if (!((vis >> j) & 1)) t[j] = -CUDART_INF_F;
        }
        float mx = t[0];
#pragma unroll
        for (int j = 1; j < NK; j++) mx = fmaxf(mx, t[j]);
        mx *= rs;
        float f = 1.0f;  // O's factor
        if (mx > m + GROW) {
          l *= ex2(m - mx);
          const float g = inv * ex2(mx - m);
          m = mx;
          inv = fminf(g, 0x1p100f);
          if (g > 0x1p100f) f = 0x1p100f / g;
        }
        const float mu = m == -CUDART_INF_F ? 0.0f : m;
        const float2 rs2 = make_float2(rs, rs), mu2 = make_float2(-mu, -mu);
        float2 sum = make_float2(0.0f, 0.0f);
#pragma unroll
        for (int j = 0; j < NK / 2; j++) {
          t2[j] = fma2(t2[j], rs2, mu2);
          t2[j].x = ex2(t2[j].x);
          t2[j].y = ex2(t2[j].y);
          sum = add2(sum, t2[j]);
        }
        l += sum.x + sum.y;
        float top = ex2(mx - mu) * vmax;  // at least the largest weight times scale
        if (each) {
          top = 0.0f;
#pragma unroll
          for (int j = 0; j < NK / 4; j++) {
            const float4 d = dv4[j];
            const float dd[4] = {d.x, d.y, d.z, d.w};
#pragma unroll
            for (int e = 0; e < 4; e++) {
              t[4 * j + e] = (vis >> (4 * j + e)) & 1 ? t[4 * j + e] * dd[e] : 0.0f;
              top = fmaxf(top, t[4 * j + e]);
            }
          }
        }
        if (top * inv > TOP) {
          const float now = SET / fmaxf(top, 0x1p-100f);
          f *= now / inv;
          inv = now;
        }
        if (__any_sync(0xffffffffu, f != 1.0f)) scale_o(i, f);
        const float2 inv2 = make_float2(inv, inv);
        if (i > 0) wait(pvdone, (i - 1) & 1, abort);  // P's memory is free
#pragma unroll
        for (int c = 0; c < NK / 8; c++) {
          uint32_t w[4];
#pragma unroll
          for (int j = 0; j < 2; j++) {
            float2 x0 = mul2(t2[4 * c + 2 * j], inv2), x1 = mul2(t2[4 * c + 2 * j + 1], inv2);
            if (!each) {
              const float4 d = dv4[2 * c + j];
              x0 = mul2(x0, make_float2(d.x, d.y));
              x1 = mul2(x1, make_float2(d.z, d.w));
            }
            w[2 * j] = pack2(x0.x, x0.y);
            w[2 * j + 1] = pack2(x1.x, x1.y);
          }
          sts128(sb + L::P + c * (ROWS * 16) + tid * 16, w[0], w[1], w[2], w[3]);
        }
        fence_async_smem();
      } else if (i > 0) {
        wait(pvdone, (i - 1) & 1, abort);  // else a warp without rows could arrive twice in one phase
      }
      tc_fence_before();
      mbar_arrive(pready);
    }
    // ---- the rows
    if (nt > 0) wait(pvdone, (nt - 1) & 1, abort);
    tc_fence_after();
    if (work) {
      const int i = tok, h = u.h * a.group + (min(row, u.rows - 1) - i * a.group);
      const long long at = u.sv.first + i;
      const bool on = row < u.rows, part = u.nch > 1;
      float f = 1.0f / inv;
      if (*abort) f = l = CUDART_NAN_F;
      if (part) {
        if (on) a.part_ml[(at * a.q.n_head + h) * a.n_chunk + u.ch] = make_float2(m, l);
      } else {
        f *= l > 0.0f || isnan(l) ? 1.0f / l : 0.0f;
      }
      if (l == 0.0f) f = 0.0f;
      float *po = part ? a.part_o + ((at * a.q.n_head + h) * a.n_chunk + u.ch) * DH : nullptr;
      const long long off = at * a.q.out_tok_stride + (long long)h * a.q.out_head_stride;
#pragma unroll
      for (int c = 0; c < DH / 32; c++) {
        float v[32];
        if (nt > 0) {
          ld32(tmem + lanes + L::O_COL + 32 * c, v);
        } else {
#pragma unroll
          for (int j = 0; j < 32; j++) v[j] = 0.0f;
        }
        if (!on) continue;
#pragma unroll
        for (int k = 0; k < 4; k++) {
          float x[8];
#pragma unroll
          for (int j = 0; j < 8; j++) x[dim8<TYPE>(j)] = f == 0.0f ? 0.0f : v[8 * k + j] * f;
          const int d0 = 32 * c + 8 * k;
          if (part) store_n<float, 8>(po + d0, true, x);
          else if (a.q.type == T_F16) store_n<__half, 8>(reinterpret_cast<__half *>(a.q.out) + off + d0, a.vec_o, x);
          else store_n<__nv_bfloat16, 8>(reinterpret_cast<__nv_bfloat16 *>(a.q.out) + off + d0, a.vec_o, x);
        }
      }
    }
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 4) {
    tc_fence_after();
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(L::COLS) : "memory");
  }
}

}  // namespace

cudaError_t launch_kv_attn_tc(const AttnKArgs &a, unsigned blocks, cudaStream_t st) {
  void (*k)(AttnKArgs) = a.c.type == PK_KV_Q8 ? (a.c.head_dim == 64 ? k_kv_attn_tc<PK_KV_Q8, 64> : k_kv_attn_tc<PK_KV_Q8, 128>)
                                              : (a.c.head_dim == 64 ? k_kv_attn_tc<PK_KV_Q4, 64> : k_kv_attn_tc<PK_KV_Q4, 128>);
  const int smem = a.c.head_dim == 64 ? Lay<64>::BYTES : Lay<128>::BYTES;
  const cudaError_t e = cudaFuncSetAttribute(k, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
  if (e != cudaSuccess) return e;
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(blocks);
  cfg.blockDim = dim3(SOFT + CONV);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = st;
  cudaLaunchAttribute at{};
  at.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  at.val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = &at;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, k, a);
}

}  // namespace pk
