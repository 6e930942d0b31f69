// pk_cache_attn_tc.cu -- attention over the quantised cache for many query
// rows of a kv head (drafted trees, prompt chunks; half-precision queries) on
// the fifth-generation tensor cores.  The formulas are pk_cache_attn.cu's.
//
// A CTA takes 128 rows (token, query head) of one kv head over one chunk of
// positions, 64 at a time: S = Q K^T (M 128 x N 64 x K head_dim) into one of
// two TMEM buffers, weights P in their place, O += P V (M 128 x N head_dim x
// K 64) in TMEM.  416 threads:
//   warps 0-3   softmax: thread = row = TMEM lane.  Scores from TMEM, the
//               scales D^K and D^V applied in f32 (two at a time), weights as
//               f16 into the scores' columns.
//   warps 4-7   K's codes, and the scales of both: a tile's are asked for a
//               tile ahead, made f16 (exact) and put into the operand's layout.
//   warps 8-11  V's codes.
//   warp 12     issues the products.
// Two CTAs share an SM (100 KB and 256 TMEM columns each), so that one's
// products run beside the other's softmax.  Operands are in the canonical
// layout without swizzle, core matrices of 8 rows x 16 bytes.  V's rows are
// stored as K's, which makes it an N-major operand.
//
// A row keeps one reference m for its weights 2^(s - m): they are summed as
// they are and multiplied by D^V into f16.  It is set so that the row's
// largest product is 2^6 (f16 ends at 2^16) and stays until a tile's weights
// could pass f16, which their sum tells, being at least the largest: most
// tiles need no maximum and leave O as it is.  A tile that does, the first
// one, and those with masked positions take the long way: the largest score,
// the largest product, a new reference if needed, the sums and O scaled by
// 2^(old - new).
//
// Every wait is bounded: one that runs out sets the CTA's abort flag, after
// which no wait waits, and its rows are written as NaN.
#include <algorithm>

#include "pk_cache_attn.cuh"
#include "pk_launch.h"
#include "pk_tcgen05.cuh"

namespace pk {
namespace {

constexpr int NK = 64;                      // positions a tile
constexpr int ROWS = TC_ATTN_ROWS;
constexpr int SOFT = 128, CONV = 128, THREADS = SOFT + 2 * CONV + 32;
// Registers: two CTAs an SM leave 72 a thread; the code warps' share of them
// goes to the softmax's.
constexpr int REGS = 72, REGS_SOFT = 112, REGS_CONV = 48;
static_assert(SOFT * REGS_SOFT + 2 * CONV * REGS_CONV + 32 * REGS <= THREADS * REGS, "no more than the launch's");
static_assert(2 * THREADS * REGS <= 65536, "two CTAs an SM");
constexpr unsigned long long WAIT_NS = 2000000000ull;

template <int DH>
struct Lay {
  // chunks of 16 bytes (8 dimensions) of consecutive positions; one chunk's
  // stride is 16 bytes more than its 64 positions, so that the 16 lanes that
  // store a position's chunks touch every bank once
  static constexpr int CH = NK * 16 + 16, TILE = DH / 8 * CH;
  static constexpr int Q = 0, K = Q + ROWS * DH * 2, V = K + 2 * TILE, SC = V + 2 * TILE;
  // of four tiles: D^K [NK], D^V [NK]; positions that hold something (2 words), largest D^V of 32 (2)
  static constexpr int SCB = 2 * NK * 4 + 16, BAR = SC + 4 * SCB, ML = BAR + 112, BYTES = ML + ROWS * 8;
  static_assert(ROWS * (DH + 4) * 4 <= SC, "a cluster's sums take the operands' place");
  static constexpr int S_COL = 0, O_COL = 2 * NK, COLS = 256;
};

// Waits for phase `parity` of mbarrier bar; called by whole warps, whose lanes
// leave it together (tcgen05 loads and stores are the whole warp's).
__device__ __forceinline__ void wait(uint32_t bar, uint32_t parity, volatile int *abort) {
  if (!mbar_test(bar, parity)) {
    const unsigned long long t0 = gtime_ns();
    while (!mbar_test(bar, parity) && !*abort)
      if (gtime_ns() - t0 > WAIT_NS) *abort = 1;
  }
  __syncwarp();
}

// This warpgroup's registers a thread from here on.
template <bool MORE, int N>
__device__ __forceinline__ void set_regs() {
  if (MORE) asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(N));
  else asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(N));
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
// The same with A in TMEM (f16, two a column).
template <int N, bool BMN>
__device__ __forceinline__ void mma_f16_ts(uint32_t d, uint32_t a, uint64_t b, bool acc) {
  constexpr uint32_t idesc = (1u << 4) | ((BMN ? 1u : 0u) << 16) | ((uint32_t)(N >> 3) << 17) | ((uint32_t)(128 >> 4) << 24);
  asm volatile(
      "{\n .reg .pred p, e;\n elect.sync _|e, 0xffffffff;\n setp.ne.b32 p, %4, 0;\n"
      " @e tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, {%5, %6, %7, %8}, p;\n}" ::"r"(d),
      "r"(a), "l"(b), "r"(idesc), "r"((uint32_t)acc), "r"(0), "r"(0), "r"(0), "r"(0)
      : "memory");
}
// 16 and 32 consecutive TMEM columns of this thread's lane.
__device__ __forceinline__ void ld16(uint32_t t, float (&v)[16]) {
  asm volatile("tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];\n tcgen05.wait::ld.sync.aligned;"
               : "=f"(v[0]), "=f"(v[1]), "=f"(v[2]), "=f"(v[3]), "=f"(v[4]), "=f"(v[5]), "=f"(v[6]), "=f"(v[7]), "=f"(v[8]), "=f"(v[9]), "=f"(v[10]), "=f"(v[11]), "=f"(v[12]), "=f"(v[13]), "=f"(v[14]), "=f"(v[15])
               : "r"(t)
               : "memory");
}
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
__device__ __forceinline__ void st16(uint32_t t, const uint32_t (&v)[16]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16};" ::"r"(t),
      "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7]), "r"(v[8]), "r"(v[9]), "r"(v[10]), "r"(v[11]), "r"(v[12]), "r"(v[13]), "r"(v[14]), "r"(v[15])
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
__global__ void __launch_bounds__(THREADS, 2) k_kv_attn_tc(const AttnKArgs a) {
  using L = Lay<DH>;
  constexpr int RB = TYPE == PK_KV_Q8 ? DH : DH / 2, SW = TYPE == PK_KV_Q8 ? 1 : 2;
  extern __shared__ __align__(1024) uint8_t smem[];
  pdl_wait();
  const Unit u = unit_of(a);
  const int tile0 = u.rt * ROWS;
  const bool cluster = a.cluster && u.nch > 1;
  if (tile0 >= u.rows || (u.ch >= max(u.nch, 1) && !cluster)) {
    pdl_trigger();
    return;
  }
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const uint32_t sb = shaddr(smem);
  // barriers: S full x 2, K and scales ready x 4, P ready x 2, PV done x 2, V ready x 2; the TMEM address; the abort flag
  const uint32_t bar = sb + L::BAR, sfull = bar, kready = bar + 16, pready = bar + 48, pvdone = bar + 64, vready = bar + 80;
  volatile int *abort = reinterpret_cast<volatile int *>(smem + L::BAR + 100);
  if (tid == 0) {
    mbar_init(sfull, 2);  // the products, and the warp that issues them (which has seen the scales)
    mbar_init(sfull + 8, 2);
    for (int i = 0; i < 4; i++) mbar_init(kready + 8 * i, CONV);
    mbar_init(pready, SOFT);
    mbar_init(pready + 8, SOFT);
    mbar_init(vready, CONV);
    mbar_init(vready + 8, CONV);
    mbar_init(pvdone, 1);
    mbar_init(pvdone + 8, 1);
    *abort = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (warp == 12) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(bar + 96), "r"(L::COLS) : "memory");
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
  const uint32_t tmem = *reinterpret_cast<volatile uint32_t *>(smem + L::BAR + 96);
  // without a mask nobody sees past the tile's last token
  const int last = (min(tile0 + ROWS, u.rows) - 1) / a.group;
  const int hi = a.q.mask ? u.hi : min(u.hi, u.sv.ctx + last + 1);
  const int nt = hi > u.lo ? (hi - u.lo + NK - 1) / NK : 0;

  if (warp == 12) {  // ---------------------------------------------- products
    auto scores = [&](int i) {
      wait(kready + 8 * (i & 3), (i >> 2) & 1, abort);
      tc_fence_after();
      // (addresses made anew each time: kept across the loop, the descriptors
      // alone would take most of the registers)
      uint32_t q = sb + L::Q, k = sb + L::K + (i & 1) * L::TILE, dt = tmem + L::S_COL + (i & 1) * NK;
      asm volatile("" : "+r"(q), "+r"(k), "+r"(dt));
#pragma unroll
      for (int s = 0; s < DH / 16; s++)
        mma_f16<NK, false>(dt, tc_desc(q + s * 2 * (ROWS * 16), ROWS * 16, 128), tc_desc(k + s * 2 * L::CH, L::CH, 128), s > 0);
      if (lane == 0) mbar_arrive(sfull + 8 * (i & 1));
      __syncwarp();
      tc_commit(sfull + 8 * (i & 1));
    };
    if (nt > 0) scores(0);
    for (int i = 0; i < nt; i++) {
      if (i + 1 < nt) scores(i + 1);  // (into the columns of tile i - 1's weights: products are done in order)
      wait(vready + 8 * (i & 1), (i >> 1) & 1, abort);
      wait(pready + 8 * (i & 1), (i >> 1) & 1, abort);
      tc_fence_after();
      uint32_t w = tmem + L::S_COL + (i & 1) * NK, v = sb + L::V + (i & 1) * L::TILE;
      asm volatile("" : "+r"(w), "+r"(v));
#pragma unroll
      for (int s = 0; s < NK / 16; s++)
        mma_f16_ts<DH, true>(tmem + L::O_COL, w + s * 8, tc_desc(v + s * 16 * 16, 128, L::CH), i > 0 || s > 0);
      tc_commit(pvdone + 8 * (i & 1));
    }
  } else if (tid >= SOFT) {  // ---------------------------------------- codes
    // 16 bytes of a row a lane (RL lanes a row), NP passes of RP rows; a
    // thread's row of pass w is w * RP + ct / RL.
    set_regs<false, REGS_CONV>();
    constexpr int RL = RB / 16, RP = CONV / RL, NP = NK / RP;
    const bool is_v = warp >= 8;
    const int ct = (tid - SOFT) & (CONV - 1), sub = ct % RL, key0 = ct / RL;
    const int key = ct & (NK - 1), half = ct >> 6;  // whose scale this thread passes on (half 0: K's, 1: V's)
    static_assert(RP % 16 == 0, "a pass has whole groups of 16 rows");
    uint4 raw[NP];  // the next tile's codes and sub-scales
    uint32_t subs[TYPE == PK_KV_Q4 ? NP : 1];
    float d = 0.0f;
    bool on = false;
    // Lane x of every warp holds, for the next 8 tiles, the cache rows of
    // positions 16 (x & 3) .. of tile x >> 2, in units of 16 rows (a page is 16
    // positions or more): -1 where there is no page.  Such rows are read from
    // the cache's first, whose codes are as good as any (their scales are 0).
    int rows16 = -1;
    const uint8_t *codes = reinterpret_cast<const uint8_t *>(is_v ? a.c.v : a.c.k) + (key0 & 15) * RB + 16 * sub;
    const uint8_t *scales = reinterpret_cast<const uint8_t *>(is_v ? a.c.vs : a.c.ks) + ((key0 & 15) * SW + 1) * 4;
    const uint8_t *dp = reinterpret_cast<const uint8_t *>(half ? a.c.vs : a.c.ks) + (key & 15) * SW * 4;
    auto ask = [&](int i) {
      if (!(i & 7)) {
        const int p = u.lo + NK * (i + (lane >> 2)) + 16 * (lane & 3), j = p >> a.page_shift;
        const int pg = p < hi && j < a.s.max_pages ? __ldg(a.s.pages + (size_t)u.s * a.s.max_pages + j) : -1;
        rows16 = pg >= 0 && pg < a.c.n_pages
                     ? (int)((((long long)pg * a.c.n_kv + u.h) * a.c.page_size + (p & (a.c.page_size - 1))) >> 4)
                     : -1;
      }
#pragma unroll
      for (int w = 0; w < NP; w++) {
        const uint32_t r = max(__shfl_sync(0xffffffffu, rows16, 4 * (i & 7) + w * (RP / 16) + key0 / 16), 0);
        raw[w] = __ldg(reinterpret_cast<const uint4 *>(codes + (size_t)r * (16 * RB)));
        if (TYPE == PK_KV_Q4) subs[w] = __ldg(reinterpret_cast<const uint32_t *>(scales + (size_t)r * (16 * SW * 4)));
      }
      if (!is_v) {
        const int r = __shfl_sync(0xffffffffu, rows16, 4 * (i & 7) + key / 16);
        on = r >= 0 && u.lo + NK * i + key < hi;
        d = __ldg(reinterpret_cast<const float *>(dp + (size_t)max(r, 0) * (16 * SW * 4)));
      }
    };
    auto put = [&](uint32_t dst) {
#pragma unroll
      for (int w = 0; w < NP; w++) {
        const uint4 x = raw[w];
        const uint32_t at = dst + (w * RP + key0) * 16;
        if (TYPE == PK_KV_Q8) {
          // two chunks of 8 dimensions; half the lanes of a row begin with the
          // second, so that eight lanes' stores touch every bank once
          const bool swap = sub >= RL / 2;
          const uint32_t a0 = swap ? x.z : x.x, a1 = swap ? x.w : x.y, b0 = swap ? x.x : x.z, b1 = swap ? x.y : x.w;
          const uint32_t ca = at + (2 * sub + swap) * L::CH, cb = at + (2 * sub + !swap) * L::CH;
          sts128(ca, codes_of(a0, 0x4140), codes_of(a0, 0x4342), codes_of(a1, 0x4140), codes_of(a1, 0x4342));
          sts128(cb, codes_of(b0, 0x4140), codes_of(b0, 0x4342), codes_of(b1, 0x4140), codes_of(b1, 0x4342));
        } else {  // four chunks, one sub-scale
          const int s = (int)((subs[w] >> (4 * sub)) & 15u);
          const uint32_t s2 = dup_h(s), m2 = dup_h(-1032 * s), y[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
          for (int c = 0; c < 4; c++)
            sts128(at + (4 * sub + c) * L::CH, nibbles_of(y[c], s2, m2), nibbles_of(y[c] >> 4, s2, m2), nibbles_of(y[c] >> 8, s2, m2),
                   nibbles_of(y[c] >> 12, s2, m2));
        }
      }
    };
    // both scales of tile i and the tile's summary, in place of tile i - 4's:
    // tile i - 2's scores are full, so tile i - 4's weights have been used
    auto put_scales = [&](int i) {
      uint8_t *sc = smem + L::SC + (i & 3) * L::SCB;
      reinterpret_cast<float *>(sc)[half * NK + key] = on ? d : 0.0f;
      if (half == 0) {
        const unsigned m = __ballot_sync(0xffffffffu, on);
        if (lane == 0) reinterpret_cast<uint32_t *>(sc + 2 * NK * 4)[key >> 5] = m;
      } else {
        const uint32_t x = __reduce_max_sync(0xffffffffu, on ? __float_as_uint(d) & 0x7fffffffu : 0);
        if (lane == 0) reinterpret_cast<uint32_t *>(sc + 2 * NK * 4 + 8)[key >> 5] = x;
      }
    };
    if (nt > 0) ask(0);
    for (int i = 0; i < nt; i++) {
      // K's buffer is free once tile i - 2's scores are there, V's once its
      // products with V are
      if (i >= 2) wait((is_v ? pvdone : sfull) + 8 * (i & 1), ((i - 2) >> 1) & 1, abort);
      put(sb + (is_v ? L::V : L::K) + (i & 1) * L::TILE);
      if (!is_v) put_scales(i);
      fence_async_smem();
      mbar_arrive(is_v ? vready + 8 * (i & 1) : kready + 8 * (i & 3));
      if (i + 1 < nt) ask(i + 1);
    }
    set_regs<true, REGS>();
  } else {  // ------------------------------------------------------------ softmax
    set_regs<true, REGS_SOFT>();
    const uint32_t lanes = (uint32_t)(warp * 32) << 16;
    const bool work = tile0 + warp * 32 < u.rows;  // (the whole warp)
    const int tok = min(row, u.rows - 1) / a.group;
    float m = -CUDART_INF_F, l = 0.0f;
    const float2 rs2 = make_float2(rs, rs);
    auto pv_wait = [&](int i) { wait(pvdone + 8 * (i & 1), (i >> 1) & 1, abort); };
    // O's row times f, once the products before are done (i > 0)
    auto scale_o = [&](int i, float f) {
      if (i == 0) return;
      pv_wait(i - 1);
      tc_fence_after();
#pragma unroll 1
      for (int c = 0; c < DH / 16; c++) {
        float v[16];
        __syncwarp();
        ld16(tmem + lanes + L::O_COL + 16 * c, v);
#pragma unroll
        for (int j = 0; j < 16; j++) v[j] *= f;
        st16(tmem + lanes + L::O_COL + 16 * c, reinterpret_cast<const uint32_t(&)[16]>(v));
      }
    };
    for (int i = 0; i < nt; i++) {
      const int b = i & 1, p0 = u.lo + NK * i;
      wait(sfull + 8 * b, (i >> 1) & 1, abort);
      tc_fence_after();
      if (work) {
        const uint8_t *sc = smem + L::SC + (i & 3) * L::SCB;
        const float4 *dk4 = reinterpret_cast<const float4 *>(sc), *dv4 = reinterpret_cast<const float4 *>(sc + NK * 4);
        const uint4 r4 = *reinterpret_cast<const uint4 *>(sc + 2 * NK * 4);
        const uint64_t held = (uint64_t)r4.y << 32 | r4.x;
        const float vmax = fmaxf(__uint_as_float(r4.z), __uint_as_float(r4.w));
        const bool masked = p0 + NK > min(u.sv.ctx, hi) || held != ~0ull;
        const uint32_t cols = tmem + lanes + L::S_COL + NK * b;
        float t[32];
        float2 *t2 = reinterpret_cast<float2 *>(t);
        auto scores = [&](int c) {  // D^K q'.c of positions 32 c ..
          __syncwarp();
          ld32(cols + 32 * c, t);
#pragma unroll
          for (int j = 0; j < 8; j++) {
            const float4 d = dk4[8 * c + j];
            t2[2 * j] = mul2(t2[2 * j], make_float2(d.x, d.y));
            t2[2 * j + 1] = mul2(t2[2 * j + 1], make_float2(d.z, d.w));
          }
        };
        uint32_t w[2][16];
        float2 sum[2];
        auto weights = [&](int c, uint32_t seen) {  // of the scores in t
          const float2 mu2 = make_float2(-m, -m);
#pragma unroll
          for (int j = 0; j < 8; j++) {
            const float4 d = dv4[8 * c + j];
#pragma unroll
            for (int e = 0; e < 2; e++) {
              float2 x = fma2(t2[2 * j + e], rs2, mu2);
              x.x = ex2(x.x);
              x.y = ex2(x.y);
              if (seen != 0xffffffffu) {
                if (!((seen >> (4 * j + 2 * e)) & 1)) x.x = 0.0f;
                if (!((seen >> (4 * j + 2 * e + 1)) & 1)) x.y = 0.0f;
              }
              sum[e] = add2(sum[e], x);
              x = mul2(x, e ? make_float2(d.z, d.w) : make_float2(d.x, d.y));
              if (seen != 0xffffffffu) {  // (a scale that is not seen may be anything)
                if (!((seen >> (4 * j + 2 * e)) & 1)) x.x = 0.0f;
                if (!((seen >> (4 * j + 2 * e + 1)) & 1)) x.y = 0.0f;
              }
              w[c][2 * j + e] = pack2(x.x, x.y);
            }
          }
        };
        bool longer = masked;
        if (!masked) {
          sum[0] = sum[1] = make_float2(0.0f, 0.0f);
#pragma unroll
          for (int c = 0; c < 2; c++) {
            scores(c);
            weights(c, 0xffffffffu);
          }
          const float all = (sum[0].x + sum[0].y) + (sum[1].x + sum[1].y);
          longer = __any_sync(0xffffffffu, !(all * vmax <= TOP && all <= 0x1p100f));  // (m is -inf at first: infinite)
          if (!longer) l += all;
        }
        if (longer) {
          const uint64_t vis = !masked ? ~0ull : row < u.rows ? held & seen_by(a, u, tok, p0, hi) : 0;
          float mx = -CUDART_INF_F, top = 0.0f;
#pragma unroll 1
          for (int c = 0; c < 2; c++) {
            scores(c);
#pragma unroll
            for (int j = 0; j < 32; j++)
              if ((vis >> (32 * c + j)) & 1) mx = fmaxf(mx, t[j]);
          }
          mx *= rs;
          // (every lane goes through the loads from TMEM, rows that see nothing too)
          const float *dv = reinterpret_cast<const float *>(dv4);
#pragma unroll 1
          for (int c = 0; c < 2; c++) {
            scores(c);
#pragma unroll
            for (int j = 0; j < 32; j++)
              if ((vis >> (32 * c + j)) & 1) top = fmaxf(top, ex2(fmaf(t[j], rs, -mx)) * dv[32 * c + j]);
          }
          float f = 1.0f;
          const float most = mx + log2f(fmaxf(top, 0x1p-100f));  // the largest product's exponent
          if (mx != -CUDART_INF_F && (m == -CUDART_INF_F || most > m + 8.0f || mx > m + 90.0f)) {
            const float now = fmaxf(most - 6.0f, mx - 90.0f);
            f = ex2(m - now);
            l *= f;
            m = now;
          }
          if (__any_sync(0xffffffffu, f != 1.0f)) scale_o(i, f);
          sum[0] = sum[1] = make_float2(0.0f, 0.0f);
          const float keep = m;
          if (m == -CUDART_INF_F) m = 0.0f;  // (nothing seen yet: every weight is masked)
#pragma unroll
          for (int c = 0; c < 2; c++) {
            scores(c);
            weights(c, (uint32_t)(vis >> (32 * c)));
          }
          m = keep;
          l += (sum[0].x + sum[0].y) + (sum[1].x + sum[1].y);
        }
        __syncwarp();
        st16(cols, w[0]);  // the weights take their scores' columns, two a column
        st16(cols + 16, w[1]);
        asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory");
      }
      tc_fence_before();
      mbar_arrive(pready + 8 * b);
    }
    // ---- the rows
    if (nt > 0) pv_wait(nt - 1);
    tc_fence_after();
    if (work) {
      const int i = tok, h = u.h * a.group + (min(row, u.rows - 1) - i * a.group);
      const long long at = u.sv.first + i;
      const bool on = row < u.rows, part = u.nch > 1;
      float f = 1.0f;
      if (*abort) f = l = CUDART_NAN_F;
      if (part) {
        if (on && cluster) *reinterpret_cast<float2 *>(smem + L::ML + tid * 8) = make_float2(m, l);
        else if (on) a.part_ml[((at * a.q.n_head + h) * a.n_chunk) + u.ch] = make_float2(m, l);
      } else {
        f *= l > 0.0f || isnan(l) ? 1.0f / l : 0.0f;
      }
      if (l == 0.0f) f = 0.0f;
      // (in a cluster: into shared memory, where the operands were)
      float *po = !part ? nullptr : cluster ? reinterpret_cast<float *>(smem) + tid * (DH + 4) : a.part_o + ((at * a.q.n_head + h) * a.n_chunk + u.ch) * DH;
      const long long off = at * a.q.out_tok_stride + (long long)h * a.q.out_head_stride;
#pragma unroll
      for (int c = 0; c < DH / 32; c++) {
        float v[32];
        __syncwarp();
        if (nt > 0) {
          ld32(tmem + lanes + L::O_COL + 32 * c, v);
        } else {
#pragma unroll
          for (int j = 0; j < 32; j++) v[j] = 0.0f;
        }
#pragma unroll
        for (int k = 0; k < 4 && on; k++) {
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
    __syncwarp();
    set_regs<false, REGS>();
  }
  tc_fence_before();
  __syncthreads();
  if (cluster) join_cluster<DH>(a, u, tile0, ROWS, sb, sb + L::ML, THREADS);
  if (warp == 12) {
    tc_fence_after();
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(L::COLS) : "memory");
  }
}

}  // namespace

cudaError_t launch_kv_attn_tc(const AttnKArgs &a, int cluster, unsigned blocks, cudaStream_t st) {
  void (*k)(AttnKArgs) = a.c.type == PK_KV_Q8 ? (a.c.head_dim == 64 ? k_kv_attn_tc<PK_KV_Q8, 64> : k_kv_attn_tc<PK_KV_Q8, 128>)
                                              : (a.c.head_dim == 64 ? k_kv_attn_tc<PK_KV_Q4, 64> : k_kv_attn_tc<PK_KV_Q4, 128>);
  const int smem = a.c.head_dim == 64 ? Lay<64>::BYTES : Lay<128>::BYTES;
  // the split of the registers would wait forever for what a launch does not have
  static std::atomic<unsigned> checked{0};
  const unsigned bit = 1u << (2 * (a.c.type == PK_KV_Q4) + (a.c.head_dim == 128));
  if (!(checked.load(std::memory_order_relaxed) & bit)) {
    cudaFuncAttributes f;
    const cudaError_t e = cudaFuncGetAttributes(&f, reinterpret_cast<const void *>(k));
    if (e != cudaSuccess) return e;
    if (f.numRegs != REGS) return cudaErrorInvalidConfiguration;
    checked.fetch_or(bit, std::memory_order_relaxed);
  }
  return launch_cluster(k, cluster, dim3(blocks), dim3(THREADS), smem, st, a);
}

}  // namespace pk
