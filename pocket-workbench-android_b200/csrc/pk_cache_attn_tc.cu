// pk_cache_attn_tc.cu -- attention over the quantised cache for many query
// rows of a kv head (drafted trees, prompt chunks) on the fifth-generation
// tensor cores.  The formulas are pk_cache_attn.cu's.
//
// A CTA takes one or two blocks of 128 rows (token, query head) of one kv head
// over one chunk of positions, 64 at a time: S = Q K^T (M 128 x N 64 x K
// head_dim) into one of two TMEM buffers, weights P, O += P V (M 128 x N
// head_dim x K 64) in TMEM.  Warps, of a block each where it says so:
//   4 a block  softmax.  Four lanes share a row (the layout of the tensor
//              core's own fragments): a thread has 4 rows and a quarter of the
//              columns, and so reads a quarter of the tile's scales D^K and
//              D^V (with a row a thread, those reads, 512 bytes to the warp
//              however few they are, were a third of shared memory's time).
//   4          K's codes, and the scales of both: a tile's are asked for a
//              tile ahead, made f16 (exact) and put into the operand's layout.
//   4          V's codes.
//   1          issues the products.
// Half precision: one block, P as f16 in S's columns, O summed in TMEM (long
// sums in parts, added up in the scratch), and two CTAs an SM (100 KB and 256 TMEM columns each), so that one's products run
// beside the other's softmax.  f32 (head_dim 64): queries and weights are two
// f16 terms each (2^-22), and a tile's O is added to the row's sums in
// registers, because the tensor core's sums drop what they shift out; two
// blocks share a CTA's codes, one CTA an SM.  Operands are in the canonical
// layout without swizzle, core matrices of 8 rows x 16 bytes (a product takes
// 61 cycles so, 66 with 128-byte swizzle).  V's rows are stored as K's, which
// makes it an N-major operand.
//
// Measured: 8 sequences of 32000 positions with trees of 64, 64 heads over 8,
// f16, Q8: 800 to 847 us by the box, 672 to 635 TFLOP/s; 40 sequences of up to
// 15000 positions, 5 drafts each, bf16, Q4: 238 us; two prompt chunks of 509
// tokens behind up to 2900 positions, 36 heads, f32, Q8: 146 to 151 us.  What bounds it: a product of N 64
// takes as long as one of N 128, so the tensor core is busy for 830 cycles of
// the 1,400 or so that a tile of 64 positions takes an SM; 128 positions a step
// would need 384 TMEM columns a CTA.
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
// which no wait for a buffer waits, and its rows are written as NaN.  The warp
// that issues the products waits for all of them before it lets go of the
// tensor memory, flag or not.
#include <algorithm>
#include <atomic>
#include <type_traits>

#include "pk_cache_attn.cuh"
#include "pk_launch.h"
#include "pk_tcgen05.cuh"

namespace pk {
namespace {

constexpr int NK = 64;                      // positions a tile
constexpr unsigned long long WAIT_NS = 2000000000ull;
// Tiles of one sum in TMEM (half precision).  Chunks of more take the kernel's
// LONG form: its additions to the scratch cost the others 2% by their size.
template <class E>
constexpr int SUM_TILES = sum_most(std::is_same_v<E, __half> ? T_F16 : T_BF16) / NK;

// Terms of a query or weight: one f16 for half precision, two for f32.
template <class E>
constexpr int terms_of = std::is_same_v<E, float> ? 2 : 1;

// Geometry, by the terms.
template <int DH, int NT>
struct Lay {
  static constexpr int BLK = NT;  // blocks of 128 rows
  // (two blocks: whole warpgroups, as the last one gives registers away too)
  static constexpr int ROWS = 128 * BLK, SOFT = 128 * BLK, CONV = 128, MMA = BLK == 1 ? 32 : 128, THREADS = SOFT + 2 * CONV + MMA;
  // Registers a thread: at launch, and after the others have given the softmax
  // warps theirs.
  static constexpr int CTAS = BLK == 1 ? 2 : 1, REGS = BLK == 1 ? 72 : 96, REGS_SOFT = BLK == 1 ? 104 : 168;
  static constexpr int REGS_CONV = BLK == 1 ? 56 : 48, REGS_MMA = BLK == 1 ? REGS : 48;
  static_assert(SOFT * REGS_SOFT + 2 * CONV * REGS_CONV + MMA * REGS_MMA <= THREADS * REGS, "no more than the launch's");
  static_assert(CTAS * THREADS * REGS <= 65536, "all of an SM's CTAs");
  // chunks of 16 bytes (8 dimensions) of consecutive positions; one chunk's
  // stride is 16 bytes more than its 64 positions, so that the lanes that
  // store together touch every bank once
  static constexpr int CH = NK * 16 + 16, TILE = DH / 8 * CH;
  static constexpr int QT = ROWS * DH * 2;  // a term of the queries
  static constexpr int Q = 0, K = Q + NT * QT, V = K + 2 * TILE, OPS = V + 2 * TILE, SUMS = ROWS * (DH + 4) * 4;
  static constexpr int SC = OPS > SUMS ? OPS : SUMS;  // (a cluster's sums take the operands' place)
  // of four tiles: D^K [NK], D^V [NK]; positions that hold something (2 words), largest D^V of 32 (2)
  static constexpr int SCB = 2 * NK * 4 + 16, BAR = SC + 4 * SCB, ML = BAR + 64 + 48 * BLK, BYTES = ML + ROWS * 8;
  // TMEM columns of a block of 128 rows: two buffers of scores, the output;
  // f32 weights' two terms have their own, f16 ones take their scores'
  static constexpr int S_COL = 0, O_COL = 2 * NK, P_COL = O_COL + DH, COLS = 256;
  static_assert(O_COL + DH + (NT == 2 ? NK : 0) <= COLS && CTAS * BLK * COLS <= 512, "the columns there are");
};

// mbar_test that may sleep for up to 20 us: warps that ask again and again take
// issue slots from the others (prompt chunks 154 us so, 148 asleep).
__device__ __forceinline__ bool mbar_sleep(uint32_t b, uint32_t parity) {
  uint32_t ok;
  asm volatile(
      "{\n .reg .pred p;\n mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2, %3;\n selp.u32 %0, 1, 0, p;\n}"
      : "=r"(ok)
      : "r"(b), "r"(parity), "r"(20000)
      : "memory");
  return ok != 0;
}
// Waits for phase `parity` of mbarrier bar: one thread, or a whole warp, whose
// lanes leave it together (tcgen05 loads and stores are the whole warp's).
__device__ __forceinline__ void wait_one(uint32_t bar, uint32_t parity, volatile int *abort) {
  if (!mbar_sleep(bar, parity)) {
    const unsigned long long t0 = gtime_ns();
    while (!mbar_sleep(bar, parity) && !*abort)
      if (gtime_ns() - t0 > WAIT_NS) *abort = 1;
  }
}
__device__ __forceinline__ void wait(uint32_t bar, uint32_t parity, volatile int *abort) {
  wait_one(bar, parity, abort);
  __syncwarp();
}
__device__ __forceinline__ bool elect_one() {
  uint32_t one;
  asm volatile("{\n .reg .pred e;\n elect.sync _|e, 0xffffffff;\n selp.u32 %0, 1, 0, e;\n}" : "=r"(one));
  return one != 0;
}
// Signals mbarrier bar once this thread's products so far are done.
__device__ __forceinline__ void commit_one(uint32_t bar) {
  asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(bar) : "memory");
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
      "{\n .reg .pred p;\n setp.ne.b32 p, %4, 0;\n"
      " tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, {%5, %6, %7, %8}, p;\n}" ::"r"(d),
      "l"(a), "l"(b), "r"(idesc), "r"((uint32_t)acc), "r"(0), "r"(0), "r"(0), "r"(0)
      : "memory");
}
// The same with A in TMEM (f16, two a column).
template <int N, bool BMN>
__device__ __forceinline__ void mma_f16_ts(uint32_t d, uint32_t a, uint64_t b, bool acc) {
  constexpr uint32_t idesc = (1u << 4) | ((BMN ? 1u : 0u) << 16) | ((uint32_t)(N >> 3) << 17) | ((uint32_t)(128 >> 4) << 24);
  asm volatile(
      "{\n .reg .pred p;\n setp.ne.b32 p, %4, 0;\n"
      " tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, {%5, %6, %7, %8}, p;\n}" ::"r"(d),
      "r"(a), "l"(b), "r"(idesc), "r"((uint32_t)acc), "r"(0), "r"(0), "r"(0), "r"(0)
      : "memory");
}
// 16 and 32 consecutive TMEM columns of this thread's lane.
// 16 columns are asked for, and usable after wait16 (which waits for all that
// were asked for: one set at a time is in flight).
__device__ __forceinline__ void ask16(uint32_t t, float (&v)[16]) {
  asm volatile("tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];"
               : "=f"(v[0]), "=f"(v[1]), "=f"(v[2]), "=f"(v[3]), "=f"(v[4]), "=f"(v[5]), "=f"(v[6]), "=f"(v[7]), "=f"(v[8]), "=f"(v[9]), "=f"(v[10]), "=f"(v[11]), "=f"(v[12]), "=f"(v[13]), "=f"(v[14]), "=f"(v[15])
               : "r"(t));
}
__device__ __forceinline__ void wait16(float (&v)[16]) {
  asm volatile("tcgen05.wait::ld.sync.aligned;"
               : "+f"(v[0]), "+f"(v[1]), "+f"(v[2]), "+f"(v[3]), "+f"(v[4]), "+f"(v[5]), "+f"(v[6]), "+f"(v[7]), "+f"(v[8]), "+f"(v[9]), "+f"(v[10]), "+f"(v[11]), "+f"(v[12]), "+f"(v[13]), "+f"(v[14]), "+f"(v[15]));
}
__device__ __forceinline__ void ld16(uint32_t t, float (&v)[16]) {
  ask16(t, v);
  wait16(v);
}
// The same 16 columns with four lanes a row: thread (lane) holds rows lane / 4
// + 8 j of the warp's 32 (j < 4), columns 8 g + 2 (lane % 4) and the next
// (g < 2), as pairs p = 4 (j / 2) + 2 g + j % 2 of v: what the tensor core's
// own operand fragments look like.
__device__ __forceinline__ void ask_quads(uint32_t t, float (&v)[16]) {
  asm volatile("tcgen05.ld.sync.aligned.16x256b.x2.b32 {%0,%1,%2,%3,%4,%5,%6,%7}, [%8];"
               : "=f"(v[0]), "=f"(v[1]), "=f"(v[2]), "=f"(v[3]), "=f"(v[4]), "=f"(v[5]), "=f"(v[6]), "=f"(v[7])
               : "r"(t));
  asm volatile("tcgen05.ld.sync.aligned.16x256b.x2.b32 {%0,%1,%2,%3,%4,%5,%6,%7}, [%8];"
               : "=f"(v[8]), "=f"(v[9]), "=f"(v[10]), "=f"(v[11]), "=f"(v[12]), "=f"(v[13]), "=f"(v[14]), "=f"(v[15])
               : "r"(t + (16u << 16)));
}
// The first 16 of the warp's 32 rows only (j < 2), and their arrival.
__device__ __forceinline__ void ask_half(uint32_t t, float (&v)[8]) {
  asm volatile("tcgen05.ld.sync.aligned.16x256b.x2.b32 {%0,%1,%2,%3,%4,%5,%6,%7}, [%8];\n tcgen05.wait::ld.sync.aligned;"
               : "=f"(v[0]), "=f"(v[1]), "=f"(v[2]), "=f"(v[3]), "=f"(v[4]), "=f"(v[5]), "=f"(v[6]), "=f"(v[7])
               : "r"(t)
               : "memory");
}
__device__ __forceinline__ void st_quads(uint32_t t, const float (&v)[16]) {
  asm volatile("tcgen05.st.sync.aligned.16x256b.x2.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8};" ::"r"(t), "f"(v[0]), "f"(v[1]), "f"(v[2]), "f"(v[3]), "f"(v[4]), "f"(v[5]), "f"(v[6]), "f"(v[7])
               : "memory");
  asm volatile("tcgen05.st.sync.aligned.16x256b.x2.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8};" ::"r"(t + (16u << 16)), "f"(v[8]), "f"(v[9]), "f"(v[10]), "f"(v[11]), "f"(v[12]), "f"(v[13]), "f"(v[14]), "f"(v[15])
               : "memory");
}
// 16 columns of f16 pairs: a thread's pairs of columns above, in order of
// groups of 8, rows lane / 4 + 8 j and the next: v of rows j < 2, u of j >= 2.
__device__ __forceinline__ void st_pairs(uint32_t t, const uint32_t *v, const uint32_t *u) {
  asm volatile("tcgen05.st.sync.aligned.16x128b.x4.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8};" ::"r"(t), "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7])
               : "memory");
  asm volatile("tcgen05.st.sync.aligned.16x128b.x4.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8};" ::"r"(t + (16u << 16)), "r"(u[0]), "r"(u[1]), "r"(u[2]), "r"(u[3]), "r"(u[4]), "r"(u[5]), "r"(u[6]), "r"(u[7])
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

// This thread's query row into the operand, f16 as it is, others scaled to
// |q'| < 2 and rounded to f16 (bf16: exact down to 2^-24 of the row's largest;
// f32: a second term holds the rest); its scale (the D^K that the row meets
// have log2(e) * scale in them).
template <int TYPE, int DH, class E>
__device__ __forceinline__ float put_q(const AttnKArgs &a, const Unit &u, int row, uint32_t dst, int stride, int term) {
  constexpr bool F16 = std::is_same_v<E, __half>;
  const bool on = row < u.rows;
  const int i = row / a.group, h = u.h * a.group + row - i * a.group;
  const E *p = reinterpret_cast<const E *>(a.q.q) + (on ? (long long)(u.sv.first + i) * a.q.q_tok_stride + (long long)h * a.q.q_head_stride : 0);
  float m = 0.0f;
  if (!F16 && on) {
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
    uint32_t w[4] = {0, 0, 0, 0}, rest[4] = {0, 0, 0, 0};
    if (on) {
      float x[8];
      load_n<E, 8>(p + 8 * c, a.vec_q, x);
#pragma unroll
      for (int j = 0; j < 4; j++) {
        const float x0 = inf_nan(x[dim8<TYPE>(2 * j)]) * down, x1 = inf_nan(x[dim8<TYPE>(2 * j + 1)]) * down;
        w[j] = pack2(x0, x1);
        if (terms_of<E> == 2) rest[j] = rest2(x0, x1, w[j]);
      }
    }
    sts128(dst + c * stride, w[0], w[1], w[2], w[3]);
    if (terms_of<E> == 2) sts128(dst + term + c * stride, rest[0], rest[1], rest[2], rest[3]);
  }
  return up;
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

template <int TYPE, int DH, class E, bool LONG>
__global__ void __launch_bounds__(Lay<DH, terms_of<E>>::THREADS, Lay<DH, terms_of<E>>::CTAS) k_kv_attn_tc(const AttnKArgs a) {
  constexpr int NT = terms_of<E>, BLK = NT;
  using L = Lay<DH, NT>;
  constexpr int ROWS = L::ROWS, SOFT = L::SOFT, CONV = L::CONV, THREADS = L::THREADS, WS = SOFT / 32;
  constexpr bool F16 = std::is_same_v<E, __half>;
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
  // barriers: K and scales ready x 4, V ready x 2; the TMEM address, the abort
  // flag; all products done; for each block of 128 rows: S full x 2, P ready x 2, PV done x 2
  const uint32_t bar = sb + L::BAR, kready = bar, vready = bar + 32, done = bar + 56, blocks = bar + 64;
  volatile int *abort = reinterpret_cast<volatile int *>(smem + L::BAR + 52);
  const int nblk = BLK == 1 ? 1 : min(BLK, (u.rows - tile0 + 127) / 128);  // that have rows
  auto sfull_of = [&](int blk, int i) { return blocks + 48 * blk + 8 * (i & 1); };
  auto pready_of = [&](int blk, int i) { return blocks + 48 * blk + 16 + 8 * (i & 1); };
  auto pvdone_of = [&](int blk, int i) { return blocks + 48 * blk + 32 + 8 * (i & 1); };
  if (tid == 0) {
    for (int i = 0; i < 4; i++) mbar_init(kready + 8 * i, CONV);
    for (int i = 0; i < 2; i++) {
      mbar_init(vready + 8 * i, CONV);
      for (int m = 0; m < BLK; m++) {
        mbar_init(sfull_of(m, i), 2);  // the products, and the warp that issues them (which has seen the scales)
        mbar_init(pready_of(m, i), 128);
        mbar_init(pvdone_of(m, i), 1);
      }
    }
    mbar_init(done, 1);
    *abort = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (warp == WS + 8) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(bar + 48), "r"(BLK * L::COLS) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  const int row = tile0 + tid;
  float rs = 0.0f;
  if (tid < SOFT) {
    rs = put_q<TYPE, DH, E>(a, u, row, sb + L::Q + tid * 16, ROWS * 16, L::QT);
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

  if (warp >= WS + 8) {  // ------------------------------------------- products
    if (BLK > 1) set_regs<false, L::REGS_MMA>();
    // one thread issues them all
    if (warp == WS + 8 && elect_one()) {
      const uint64_t qd = tc_desc(sb + L::Q, ROWS * 16, 128), kd = tc_desc(sb + L::K, L::CH, 128), vd = tc_desc(sb + L::V, 128, L::CH);
      auto scores = [&](int i) {
        wait_one(kready + 8 * (i & 3), (i >> 2) & 1, abort);
        tc_fence_after();
        for (int m = 0; m < nblk; m++) {
          const uint64_t q = qd + m * 128, k = kd + (i & 1) * (L::TILE / 16);
          const uint32_t dt = tmem + m * L::COLS + L::S_COL + (i & 1) * NK;
#pragma unroll
          for (int n = NT - 1; n >= 0; n--)  // (the smaller term first)
#pragma unroll
            for (int s = 0; s < DH / 16; s++)
              mma_f16<NK, false>(dt, q + (n * L::QT / 16 + s * 2 * ROWS), k + s * 2 * (L::CH / 16), s > 0 || n < NT - 1);
          mbar_arrive(sfull_of(m, i));
          commit_one(sfull_of(m, i));
        }
      };
      if (nt > 0) scores(0);
      for (int i = 0; i < nt; i++) {
        if (i + 1 < nt) scores(i + 1);  // (into the columns of tile i - 1's weights: products are done in order)
        wait_one(vready + 8 * (i & 1), (i >> 1) & 1, abort);
        for (int m = 0; m < nblk; m++) {
          wait_one(pready_of(m, i), (i >> 1) & 1, abort);
          tc_fence_after();
          const uint32_t w = tmem + m * L::COLS + (NT == 2 ? L::P_COL : L::S_COL + (i & 1) * NK), o = tmem + m * L::COLS + L::O_COL;
          const uint64_t v = vd + (i & 1) * (L::TILE / 16);
#pragma unroll
          for (int n = NT - 1; n >= 0; n--)
#pragma unroll
            for (int s = 0; s < NK / 16; s++)
              mma_f16_ts<DH, true>(o, w + n * (NK / 2) + s * 8, v + s * 16, (NT == 1 && (LONG ? i % SUM_TILES<E> != 0 : i > 0)) || s > 0 || n < NT - 1);
          commit_one(pvdone_of(m, i));
        }
      }
      // the operands and the tensor memory are theirs until they are done, also
      // where a wait ran out and nobody waited for them
      commit_one(done);
      const unsigned long long t0 = gtime_ns();
      while (!mbar_sleep(done, 0))
        if (gtime_ns() - t0 > WAIT_NS) {
          *abort = 1;
          break;
        }
    }
    __syncwarp();
  } else if (tid >= SOFT) {  // ---------------------------------------- codes
    // 16 bytes of a row a lane (RL lanes a row), NP passes of RP rows; a
    // thread's row of pass w is w * RP + key0.  Eight lanes that store together
    // have RS parts of a row and 8 / RS rows, so that they touch every bank
    // once (a part's chunks are 2 or 4 strides from the next part's).
    set_regs<false, L::REGS_CONV>();
    // (one body for both: two cost 15% by their size alone, the SM's warps being
    // in all parts of the loops at once)
    const bool is_v = warp >= WS + 4;
    constexpr int RL = RB / 16, RP = CONV / RL, NP = NK / RP;
    constexpr int RS = TYPE == PK_KV_Q8 ? 4 : 2;
    const int ct = (tid - SOFT) & (CONV - 1);
    const int sub = RL <= RS ? ct % RL : ct % RS + (ct / 8 % (RL / RS)) * RS;
    const int key0 = RL <= RS ? ct / RL : ct / RS % (8 / RS) + ct / (8 * RL / RS) * (8 / RS);
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
    // All are read past L1: a prompt's chunks run in streams of their own, and
    // while one stores rows, which this launch waits for, another's attention may
    // have brought their lines, with the rows as they were, into this SM's L1.
    int rows16 = -1;
    const uint8_t *codes = reinterpret_cast<const uint8_t *>(is_v ? a.c.v : a.c.k);
    const uint32_t *subs_of = reinterpret_cast<const uint32_t *>(is_v ? a.c.vs : a.c.ks);
    const float *d_of = half ? a.c.vs : a.c.ks;
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
        raw[w] = __ldcg(reinterpret_cast<const uint4 *>(codes + ((size_t)r * (16 * RB) + ((key0 & 15) * RB + 16 * sub))));
        if (TYPE == PK_KV_Q4) subs[w] = __ldcg(subs_of + ((size_t)r * (16 * SW) + ((key0 & 15) * SW + 1)));
      }
      if (!is_v) {
        const int r = __shfl_sync(0xffffffffu, rows16, 4 * (i & 7) + key / 16);
        on = r >= 0 && u.lo + NK * i + key < hi;
        d = __ldcg(d_of + ((size_t)max(r, 0) * (16 * SW) + (key & 15) * SW));
      }
    };
    auto put = [&](uint32_t dst) {
#pragma unroll
      for (int w = 0; w < NP; w++) {
        const uint4 x = raw[w];
        const uint32_t at = dst + (w * RP + key0) * 16;
        if (TYPE == PK_KV_Q8) {
          // two chunks of 8 dimensions
          sts128(at + 2 * sub * L::CH, codes_of(x.x, 0x4140), codes_of(x.x, 0x4342), codes_of(x.y, 0x4140), codes_of(x.y, 0x4342));
          sts128(at + (2 * sub + 1) * L::CH, codes_of(x.z, 0x4140), codes_of(x.z, 0x4342), codes_of(x.w, 0x4140), codes_of(x.w, 0x4342));
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
      reinterpret_cast<float *>(sc)[half * NK + key] = on ? half ? d : fminf(fmaxf(d * (a.q.scale * kLog2e), -3e38f), 3e38f) : 0.0f;  // (finite: a query may be 0)
      if (half == 0) {
        const unsigned m = __ballot_sync(0xffffffffu, on);
        if (lane == 0) reinterpret_cast<uint32_t *>(sc + 2 * NK * 4)[key >> 5] = m;
      } else {
        const uint32_t x = __reduce_max_sync(0xffffffffu, on ? __float_as_uint(d) & 0x7fffffffu : 0);
        if (lane == 0) reinterpret_cast<uint32_t *>(sc + 2 * NK * 4 + 8)[key >> 5] = x;
      }
    };
    const int n = a.poison ? 0 : nt;
    if (n > 0) ask(0);
    for (int i = 0; i < n; i++) {
      // K's buffer is free once tile i - 2's scores are there, V's once its
      // products with V are
      if (i >= 2)
        for (int m = 0; m < nblk; m++) wait(is_v ? pvdone_of(m, i) : sfull_of(m, i), ((i - 2) >> 1) & 1, abort);
      put(sb + (is_v ? L::V : L::K) + (i & 1) * L::TILE);
      if (!is_v) put_scales(i);
      fence_async_smem();
      mbar_arrive(is_v ? vready + 8 * (i & 1) : kready + 8 * (i & 3));
      if (i + 1 < n) ask(i + 1);
    }
  } else {  // ------------------------------------------------------------ softmax
    set_regs<true, L::REGS_SOFT>();
    const int blk = BLK == 1 ? 0 : warp >> 2;
    const uint32_t lanes = ((uint32_t)((warp & 3) * 32) << 16) + blk * L::COLS;
    const bool work = tile0 + warp * 32 < u.rows;  // (the whole warp)
    const int tok = min(row, u.rows - 1) / a.group;
    const int quad = lane & 3;
    // of rows lane / 4 + 8 j: the scale, the reference, this thread's part of the sum
    float rs4[4], m4[4], l4[4];
#pragma unroll
    for (int j = 0; j < 4; j++) {
      rs4[j] = __shfl_sync(0xffffffffu, rs, (lane >> 2) + 8 * j);
      m4[j] = -CUDART_INF_F;
      l4[j] = 0.0f;
    }
    auto pv_wait = [&](int i) { wait(pvdone_of(blk, i), (i >> 1) & 1, abort); };
    // f32: a tile's products with V are added to the rows' sums here, as the
    // tensor core's own additions cut off what they shift out; `added` tiles are
    float o[NT == 2 ? DH : 16];
    int added = 0;
    if (NT == 2) {
#pragma unroll
      for (int j = 0; j < DH; j++) o[NT == 2 ? j : 0] = 0.0f;
    }
    auto add_o = [&](int n) {  // so that n tiles are
      if (added >= n) return;  // (the same for the whole warp)
      added = n;
      pv_wait(n - 1);
      tc_fence_after();
      __syncwarp();
#pragma unroll
      for (int c = 0; c < DH / 16; c++) {
        float v[16];
        ask_quads(tmem + lanes + L::O_COL + 16 * c, v);
        wait16(v);
#pragma unroll
        for (int j = 0; j < 16; j++) o[NT == 2 ? 16 * c + j : 0] += v[j];
      }
    };
    // half precision: the sum of tiles .. i - 1 is added to what the scratch has
    // of the row, beside the reference that it was made with (16 rows at a time:
    // registers of the whole loop are few)
    auto keep_o = [&](int i) {
      pv_wait(i - 1);
      tc_fence_after();
#pragma unroll 1
      for (int half = 0; half < 2; half++) {
        const float m[2] = {half ? m4[2] : m4[0], half ? m4[3] : m4[1]};
        float *to[2];
        float g[2];
#pragma unroll
        for (int j = 0; j < 2; j++) {
          const int row = tile0 + warp * 32 + (lane >> 2) + 16 * half + 8 * j, r = min(row, u.rows - 1), t = r / a.group;
          const long long at = ((long long)(u.sv.first + t) * a.q.n_head + u.h * a.group + r - t * a.group) * a.n_chunk + u.ch;
          to[j] = a.part_o + at * DH + 2 * quad;
          const float before = i > SUM_TILES<E> ? a.part_ml[at].x : -CUDART_INF_F;
          g[j] = before == -CUDART_INF_F ? 0.0f : ex2(before - m[j]);
          __syncwarp();
          if (quad == 0 && row < u.rows) a.part_ml[at].x = m[j];
        }
#pragma unroll 1
        for (int c = 0; c < DH / 16; c++) {
          float v[8];
          __syncwarp();
          ask_half(tmem + lanes + ((uint32_t)(16 * half) << 16) + L::O_COL + 16 * c, v);
#pragma unroll
          for (int p = 0; p < 4; p++) {  // row 8 (p % 2), columns 8 (p / 2) and the next
            if (tile0 + warp * 32 + (lane >> 2) + 16 * half + 8 * (p & 1) >= u.rows) continue;
            float2 *x = reinterpret_cast<float2 *>(to[p & 1] + 16 * c + 8 * (p >> 1));
            const float2 o = make_float2(v[2 * p], v[2 * p + 1]);
            *x = i > SUM_TILES<E> ? fma2(*x, make_float2(g[p & 1], g[p & 1]), o) : o;
          }
        }
      }
    };
    // O's rows times f, once the products before are done (i > 0)
    auto scale_o = [&](int i, const float (&f)[4]) {
      if (i == 0) return;
      if constexpr (NT == 2) {
#pragma unroll
        for (int j = 0; j < DH; j++) o[j] *= f[2 * ((j >> 3) & 1) + ((j >> 1) & 1)];
      } else {
        pv_wait(i - 1);
        tc_fence_after();
#pragma unroll 1
        for (int c = 0; c < DH / 16; c++) {
          float v[16];
          __syncwarp();
          ask_quads(tmem + lanes + L::O_COL + 16 * c, v);
          wait16(v);
#pragma unroll
          for (int j = 0; j < 16; j++) v[j] *= f[2 * (j >> 3) + ((j >> 1) & 1)];
          st_quads(tmem + lanes + L::O_COL + 16 * c, v);
        }
      }
    };
    if (blk < nblk)
    for (int i = 0; i < nt; i++) {
      const int b = i & 1, p0 = u.lo + NK * i;
      wait(sfull_of(blk, i), (i >> 1) & 1, abort);
      tc_fence_after();
      if (work) {
        if (LONG && i > 0 && i % SUM_TILES<E> == 0) keep_o(i);
        const uint8_t *sc = smem + L::SC + (i & 3) * L::SCB;
        const float2 *dk2 = reinterpret_cast<const float2 *>(sc) + quad, *dv2 = dk2 + NK / 2;
        const uint4 r4 = *reinterpret_cast<const uint4 *>(sc + 2 * NK * 4);
        const uint64_t held = (uint64_t)r4.y << 32 | r4.x;
        const float vmax = fmaxf(__uint_as_float(r4.z), __uint_as_float(r4.w));
        const bool masked = p0 + NK > min(u.sv.ctx, hi) || held != ~0ull;
        const uint32_t cols = tmem + lanes + L::S_COL + NK * b;
        // columns 8 (2 k + g) + 2 quad and the next of a row's 64
        auto bits = [&](uint64_t vis, int k, int g) { return (uint32_t)(vis >> (16 * k + 8 * g + 2 * quad)); };
        // weights of the products in t, 16 columns; f16: all 64 columns' are
        // kept (their scores may be needed again), f32: those of two steps
        constexpr int WK = NT == 1 ? 4 : 2;
        uint32_t w[NT][2][4 * WK];
        float2 sum[4];
        auto weights = [&](int k0, int k1, const float (&t)[16], const float (&m)[4], const uint64_t *vis) {  // step k0 + k1
          const int k = k0 + k1;
#pragma unroll
          for (int g = 0; g < 2; g++) {
            const float2 dk = dk2[4 * (2 * k + g)], dv = dv2[4 * (2 * k + g)];
#pragma unroll
            for (int j = 0; j < 4; j++) {
              const int p = 4 * (j >> 1) + 2 * g + (j & 1), at = 2 * (2 * k1 + g) + (j & 1);
              float2 x = make_float2(t[2 * p], t[2 * p + 1]);
              x = F16 ? fma2(x, dk, make_float2(-m[j], -m[j])) : fma2(mul2(x, dk), make_float2(rs4[j], rs4[j]), make_float2(-m[j], -m[j]));
              x.x = ex2(x.x);
              x.y = ex2(x.y);
              const uint32_t seen = vis ? bits(vis[j], k, g) : 3u;
              if (vis) x.x = seen & 1 ? x.x : 0.0f, x.y = seen & 2 ? x.y : 0.0f;
              sum[j] = add2(sum[j], x);
              x = mul2(x, dv);
              if (vis) x.x = seen & 1 ? x.x : 0.0f, x.y = seen & 2 ? x.y : 0.0f;  // (a scale that is not seen may be anything)
              w[0][j >> 1][at] = pack2(x.x, x.y);
              if (NT == 2) w[NT - 1][j >> 1][at] = rest2(x.x, x.y, w[0][j >> 1][at]);
            }
          }
        };
        // f32: half h of the tile's are stored, the products with those of the
        // tile before being done
        auto put_two = [&](int h) {
          add_o(i);
          __syncwarp();
#pragma unroll
          for (int n = 0; n < NT; n++) st_pairs(tmem + lanes + L::P_COL + n * (NK / 2) + 16 * h, w[n][0], w[n][1]);
        };
        bool longer = masked;
        if (!masked) {
          sum[0] = sum[1] = sum[2] = sum[3] = make_float2(0.0f, 0.0f);
          __syncwarp();
          if constexpr (NT == 1) {  // 16 columns are on their way while those before are worked on
            float t[2][16];
            ask_quads(cols, t[0]);
#pragma unroll
            for (int k = 0; k < 4; k++) {
              wait16(t[k & 1]);
              if (k < 3) ask_quads(cols + 16 * (k + 1), t[(k + 1) & 1]);
              weights(0, k, t[k & 1], m4, nullptr);
            }
          } else {
#pragma unroll 1
            for (int h = 0; h < 2; h++) {
#pragma unroll
              for (int k = 0; k < 2; k++) {
                float t[16];
                ask_quads(cols + 32 * h + 16 * k, t);
                wait16(t);
                weights(2 * h, k, t, m4, nullptr);
              }
              put_two(h);
            }
          }
          // (a thread's part of a row's sum is at least the largest of its
          // weights; m is -inf at first: infinite)
          bool over = false;
          float all[4];
#pragma unroll
          for (int j = 0; j < 4; j++) {
            all[j] = sum[j].x + sum[j].y;
            over |= !(all[j] * vmax <= TOP && all[j] <= 0x1p100f);
          }
          longer = __any_sync(0xffffffffu, over);
          if (!longer) {
#pragma unroll
            for (int j = 0; j < 4; j++) l4[j] += all[j];
          }
        }
        if (longer) {
          if (NT == 2) add_o(i);
          const uint64_t mine = !masked ? ~0ull : row < u.rows ? held & seen_by(a, u, tok, p0, hi) : 0;
          uint64_t vis[4];
          float mx[4], top[4], f[4], m[4];
#pragma unroll
          for (int j = 0; j < 4; j++) {
            vis[j] = __shfl_sync(0xffffffffu, mine, (lane >> 2) + 8 * j);
            mx[j] = -CUDART_INF_F;
            top[j] = 0.0f;
          }
          // (every lane goes through the loads from TMEM, rows that see nothing too)
          auto over_seen = [&](auto step) {
#pragma unroll 1
            for (int k = 0; k < 4; k++) {
              float t[16];
              __syncwarp();
              ask_quads(cols + 16 * k, t);
              wait16(t);
#pragma unroll
              for (int g = 0; g < 2; g++) {
                const float2 dk = dk2[4 * (2 * k + g)], dv = dv2[4 * (2 * k + g)];
#pragma unroll
                for (int j = 0; j < 4; j++) {
                  const int p = 4 * (j >> 1) + 2 * g + (j & 1);
                  const uint32_t seen = bits(vis[j], k, g);
                  if (seen & 1) step(j, t[2 * p] * dk.x, dv.x);
                  if (seen & 2) step(j, t[2 * p + 1] * dk.y, dv.y);
                }
              }
            }
          };
          auto quad_max = [](float x) {
            x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 1));
            return fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 2));
          };
          over_seen([&](int j, float x, float) { mx[j] = fmaxf(mx[j], x * rs4[j]); });
#pragma unroll
          for (int j = 0; j < 4; j++) mx[j] = quad_max(mx[j]);
          over_seen([&](int j, float x, float dv) { top[j] = fmaxf(top[j], ex2(fmaf(x, rs4[j], -mx[j])) * dv); });
          bool moved = false;
#pragma unroll
          for (int j = 0; j < 4; j++) {
            f[j] = 1.0f;
            const float most = mx[j] + log2f(fmaxf(quad_max(top[j]), 0x1p-100f));  // the largest product's exponent
            if (mx[j] != -CUDART_INF_F && (m4[j] == -CUDART_INF_F || most > m4[j] + 8.0f || mx[j] > m4[j] + 90.0f)) {
              const float now = fmaxf(most - 6.0f, mx[j] - 90.0f);
              f[j] = ex2(m4[j] - now);
              l4[j] *= f[j];
              m4[j] = now;
              moved |= f[j] != 1.0f;
            }
            m[j] = m4[j] == -CUDART_INF_F ? 0.0f : m4[j];  // (nothing seen yet: all are masked)
          }
          if (__any_sync(0xffffffffu, moved)) scale_o(i, f);
          sum[0] = sum[1] = sum[2] = sum[3] = make_float2(0.0f, 0.0f);
#pragma unroll(NT == 1 ? 4 : 1)
          for (int h = 0; h < 4 / WK; h++) {
#pragma unroll
            for (int k = 0; k < WK; k++) {
              float t[16];
              __syncwarp();
              ask_quads(cols + 16 * (WK * h + k), t);
              wait16(t);
              weights(WK * h, k, t, m, vis);
            }
            if (NT == 2) put_two(h);
          }
#pragma unroll
          for (int j = 0; j < 4; j++) l4[j] += sum[j].x + sum[j].y;
        }
        __syncwarp();
        if (NT == 1) {  // the weights take their scores' columns, two a column
          st_pairs(cols, w[0][0], w[0][1]);
          st_pairs(cols + 16, w[0][0] + (NT == 1 ? 8 : 0), w[0][1] + (NT == 1 ? 8 : 0));
        }
        asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory");
      }
      tc_fence_before();
      mbar_arrive(pready_of(blk, i));
    }
    // ---- the rows
    if (nt > 0 && blk < nblk) {
      pv_wait(nt - 1);
      if (NT == 2 && work) add_o(nt);
    }
    tc_fence_after();
    // one row a lane again
    float m = 0.0f, l = 0.0f;
#pragma unroll
    for (int j = 0; j < 4; j++) {
      float x = l4[j];
      x += __shfl_xor_sync(0xffffffffu, x, 1);
      x += __shfl_xor_sync(0xffffffffu, x, 2);
      x = __shfl_sync(0xffffffffu, x, 4 * (lane & 7));
      const float y = __shfl_sync(0xffffffffu, m4[j], 4 * (lane & 7));
      if ((lane >> 3) == j) l = x, m = y;
    }
    if constexpr (NT == 2) {
      const float ok = *abort ? CUDART_NAN_F : 1.0f;
      __syncwarp();
#pragma unroll
      for (int c = 0; c < DH / 16; c++) {
        float v[16];
#pragma unroll
        for (int j = 0; j < 16; j++) v[j] = o[16 * c + j] * ok;
        st_quads(tmem + lanes + L::O_COL + 16 * c, v);
      }
      asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory");
    }
    // (a cluster's sums take the operands' place: all blocks' products are done)
    if (BLK > 1 && cluster) asm volatile("bar.sync 1, %0;" ::"r"(SOFT) : "memory");
    if (work) {
      const int i = tok, h = u.h * a.group + (min(row, u.rows - 1) - i * a.group);
      const long long at = u.sv.first + i;
      const bool on = row < u.rows, part = u.nch > 1;
      float f = 1.0f, g = 0.0f;  // g: of what a long sum has in the scratch
      if (LONG && nt > SUM_TILES<E> && on) {
        const float before = a.part_ml[(at * a.q.n_head + h) * a.n_chunk + u.ch].x;
        g = before == -CUDART_INF_F ? 0.0f : ex2(before - m);
      }
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
      for (int c = 0; c < DH / 16; c++) {
        float v[16];
        __syncwarp();
        if (NT == 2 || nt > 0) {
          ld16(tmem + lanes + L::O_COL + 16 * c, v);
        } else {
#pragma unroll
          for (int j = 0; j < 16; j++) v[j] = 0.0f;
        }
        if (LONG && nt > SUM_TILES<E> && on) {
          const float *p = a.part_o + ((at * a.q.n_head + h) * a.n_chunk + u.ch) * DH + 16 * c;
#pragma unroll
          for (int j = 0; j < 16; j++) v[j] = fmaf(g, p[j], v[j]);
        }
#pragma unroll
        for (int k = 0; k < 2 && on; k++) {
          float x[8];
#pragma unroll
          for (int j = 0; j < 8; j++) x[dim8<TYPE>(j)] = f == 0.0f ? 0.0f : v[8 * k + j] * f;
          const int d0 = 16 * c + 8 * k;
          if (part) store_n<float, 8>(po + d0, true, x);
          else store_n<E, 8>(reinterpret_cast<E *>(a.q.out) + off + d0, a.vec_o, x);
        }
      }
    }
    __syncwarp();
    set_regs<false, L::REGS>();
  }
  tc_fence_before();
  __syncthreads();
  // Only here, after the softmax warps have had their registers and given them
  // back: taken earlier (by warps without a tile) they would be missing there.
  if (warp >= WS && (BLK > 1 || warp < WS + 8)) set_regs<true, L::REGS>();
  // Before the cluster's sums: a CTA that waited for its cluster with tensor
  // memory in hand could wait for one that waits for tensor memory, which a CTA
  // of another kernel's cluster in the same state holds.
  if (warp == WS + 8) {
    tc_fence_after();
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(BLK * L::COLS) : "memory");
  }
  __syncwarp();
  if (cluster) join_cluster<DH>(a, u, tile0, ROWS, sb, sb + L::ML, THREADS);
  if (tid == 0 && a.err && *abort) atomicCAS(a.err, 0, PK_ERR_TIMEOUT);
}

struct Kernel {
  void (*k)(AttnKArgs);
  int threads, smem, regs;
};
template <int TYPE, int DH, class E>
Kernel kernel_as(bool many) {
  using L = Lay<DH, terms_of<E>>;
  if constexpr (terms_of<E> == 1)
    if (many) return {k_kv_attn_tc<TYPE, DH, E, true>, L::THREADS, L::BYTES, L::REGS};
  return {k_kv_attn_tc<TYPE, DH, E, false>, L::THREADS, L::BYTES, L::REGS};
}
template <class E>
Kernel kernel_of(const pk_kv_cache &c, bool many) {
  if (c.head_dim == 64) return c.type == PK_KV_Q8 ? kernel_as<PK_KV_Q8, 64, E>(many) : kernel_as<PK_KV_Q4, 64, E>(many);
  if constexpr (terms_of<E> == 1) return c.type == PK_KV_Q8 ? kernel_as<PK_KV_Q8, 128, E>(many) : kernel_as<PK_KV_Q4, 128, E>(many);
  return {};
}

}  // namespace

cudaError_t launch_kv_attn_tc(const AttnKArgs &a, int cluster, unsigned blocks, cudaStream_t st) {
  const int e = a.q.type == T_F32 ? 0 : a.q.type == T_F16 ? 1 : 2;
  const bool many = e && a.chunk > sum_most(a.q.type);  // (positions; only half precision sums in TMEM)
  const Kernel k = e == 0 ? kernel_of<float>(a.c, many) : e == 1 ? kernel_of<__half>(a.c, many) : kernel_of<__nv_bfloat16>(a.c, many);
  if (!k.k) return cudaErrorInvalidValue;
  // the split of the registers would wait forever for what a launch does not have
  static std::atomic<unsigned> checked{0};
  const unsigned bit = 1u << (16 * many + e * 4 + 2 * (a.c.type == PK_KV_Q4) + (a.c.head_dim == 128));
  if (!(checked.load(std::memory_order_relaxed) & bit)) {
    cudaFuncAttributes f;
    const cudaError_t err = cudaFuncGetAttributes(&f, reinterpret_cast<const void *>(k.k));
    if (err != cudaSuccess) return err;
    if (f.numRegs != k.regs) return cudaErrorInvalidConfiguration;
    checked.fetch_or(bit, std::memory_order_relaxed);
  }
  return launch_cluster(k.k, cluster, dim3(blocks), dim3(k.threads), k.smem, st, a);
}

}  // namespace pk
