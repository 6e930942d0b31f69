// pk_cache_prefix.cu -- attention of many half-precision rows over positions that
// all of them see, a prefix that a group's sequences share, on the
// fifth-generation tensor cores.  The formulas are pk_cache_attn.cu's; the parts
// (row sums, weights' sum, reference) go to the scratch.
//
// A CTA takes 256 rows (token, query head of a kv head) in two blocks over one
// chunk of positions, 128 at a time: S = Q K^T (M 128 x N 128 x K head_dim) into
// the block's 128 TMEM columns, weights P as f16 in S's first 64, O += P V in
// another 128 (head_dim 64: 64).  That is all of an SM's tensor memory, so a
// block has one S; while its softmax works, the other block's products run, which
// follow each other as O += P V (tile i), S (tile i + 1).  Against the kernel of
// pk_cache_attn_tc.cu, two CTAs of 128 rows an SM and 64 positions a tile: a
// product of N 128 takes 65 cycles where one of N 64 takes 61, and the codes are
// made f16 once for 256 rows.  No masks: what a tile has beyond the chunk's end,
// or on pages that are none, gets -inf added to its scores.
//
// Warps: 8 softmax (4 a block, four lanes a row as there), 4 that make K's codes
// f16 and pass on both scales, 4 for V's, 4 of which one thread issues the
// products.  Waits are bounded as there: one that runs out leaves NaN rows.
//
// Measured: two prefixes of 24000 positions under 800 tokens each, 64 heads over 8
// of 128, bf16, Q8: 1.39 ms, 905 TFLOP/s (the kernel of 128 rows: 1.72 ms).  What
// bounds it: a block's tile takes its softmax warps 2,600 cycles beside the other
// block's (exponentials of both alone are 2,050) and then 1,040 of products and 700
// on the way there and back, 4,300 in all, of which the two blocks' products fill
// 2,080.  Twice the softmax warps, two for the same rows: 2.01 ms for the call, then
// 1.76 (their registers did not hold a tile's weights).  The thread that issues the
// products has few registers: with its loops unrolled they were spilled, 1.55 ms.
// One chunk of four tiles takes 43,000 cycles: 13,000 until the queries are there,
// 8,000 for the first tile, 13,000 the others, 8,000 to write the rows.  Slower: one
// arrival a warp for one a thread, a first reference from 32 positions, rows by
// bulk copies (each 3% and more of the call).  All forms spill about 100 bytes a thread.
#include <algorithm>
#include <atomic>

#include "pk_cache_tc.cuh"
#include "pk_launch.h"

namespace pk {
namespace {

constexpr int PK_N = 128, PROWS = 256;  // positions a tile, rows a CTA
constexpr int PSOFT = 256, PCONV = 128, PMMA = 128, PTHREADS = PSOFT + 2 * PCONV + PMMA, PWS = PSOFT / 32;
// registers a thread: at launch, then by warps
constexpr int PREGS = 96, PREGS_SOFT = 160, PREGS_CONV = 64, PREGS_MMA = 32;
static_assert(PSOFT * PREGS_SOFT + 2 * PCONV * PREGS_CONV + PMMA * PREGS_MMA <= PTHREADS * PREGS, "no more than the launch's");

template <int DH>
struct PLay {
  static constexpr int CH = PK_N * 16 + 16, TILE = DH / 8 * CH;  // chunks of 16 bytes (8 dimensions) of a tile's positions, padded
  static constexpr int Q = 0, K = PROWS * DH * 2, V = K + 2 * TILE, OPS = V + 2 * TILE, SUMS = PROWS * (DH + 4) * 4;
  static constexpr int SC = OPS > SUMS ? OPS : SUMS;
  // of four tiles: D^K, D^V, what is added to the scores (0 or -inf), log2 D^V; positions that hold something (4 words), largest D^V of 32 (4)
  static constexpr int SCB = 4 * PK_N * 4 + 32, BAR = SC + 4 * SCB, BYTES = BAR + 64 + 48 * 2 + 8;
  static constexpr int S_COL = 0, O_COL = PK_N, COLS = 256;  // of a block's
  static_assert(BYTES <= 227 * 1024, "an SM's");
};

// A warp's 32 query rows into the operand, as put_q_half does: eight rows at a
// time, four lanes a row (eight lanes that store together have a vector of each
// row: no bank twice); rs[j]: the scale of row lane / 4 + 8 j.
template <int TYPE, int DH, class E>
__device__ __forceinline__ void put_q_rows(const AttnKArgs &a, const Unit &u, int row0, uint32_t dst, float (&rs)[4]) {
  constexpr bool F16 = std::is_same_v<E, __half>;
  constexpr int N = DH / 32;  // vectors of 8 a lane
  const int lane = threadIdx.x & 31, part = lane >> 3;
  uint4 next[N];
  auto ask = [&](int k) {
    const int row = row0 + 8 * k + (lane & 7), i = row / a.group, h = u.h * a.group + row - i * a.group;
    const bool on = row < u.rows;
    const E *p = reinterpret_cast<const E *>(a.q.q) + (on ? (long long)(u.sv.first + i) * a.q.q_tok_stride + (long long)h * a.q.q_head_stride : 0) + part * 8;
    if (on && a.vec_q) {
#pragma unroll
      for (int c = 0; c < N; c++) next[c] = __ldg(reinterpret_cast<const uint4 *>(p + 32 * c));
    } else {
      E *y = reinterpret_cast<E *>(next);
#pragma unroll
      for (int j = 0; j < 8 * N; j++) y[j] = on ? p[j / 8 * 32 + j % 8] : from_f<E>(0.0f);
    }
  };
  ask(0);
#pragma unroll 1
  for (int k = 0; k < 4; k++) {
    uint4 raw[N];
#pragma unroll
    for (int c = 0; c < N; c++) raw[c] = next[c];
    if (k < 3) ask(k + 1);
    const E *x = reinterpret_cast<const E *>(raw);
    float m = 0.0f;
    if (!F16) {
#pragma unroll
      for (int j = 0; j < 8 * N; j++) m = fmaxf(m, fabsf(to_f(x[j])));
      m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, 8));
      m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, 16));
    }
    int e = (int)(__float_as_uint(m) >> 23) - 127;
    e = m > 0.0f ? min(max(e, -100), 126) : 0;
    const float down = __int_as_float((127 - e) << 23), up = __shfl_sync(0xffffffffu, __int_as_float((e + 127) << 23), lane >> 2);
#pragma unroll
    for (int j = 0; j < 4; j++) rs[j] = j == k ? up : rs[j];
#pragma unroll
    for (int c = 0; c < N; c++) {
      uint32_t w[4];
#pragma unroll
      for (int j = 0; j < 4; j++) {
        const float x0 = to_f(x[8 * c + dim8<TYPE>(2 * j)]), x1 = to_f(x[8 * c + dim8<TYPE>(2 * j + 1)]);
        w[j] = pack2(fmaf(x0, down, x0 - x0), fmaf(x1, down, x1 - x1));  // (infinities as NaN)
      }
      sts128(dst + (8 * k + (lane & 7)) * 16 + (part + 4 * c) * (PROWS * 16), w[0], w[1], w[2], w[3]);
    }
  }
}

template <int TYPE, int DH, class E>
__global__ void __launch_bounds__(PTHREADS, 1) k_kv_prefix(const AttnKArgs a) {
  using L = PLay<DH>;
  constexpr bool F16 = std::is_same_v<E, __half>;
  constexpr int RB = TYPE == PK_KV_Q8 ? DH : DH / 2, SW = TYPE == PK_KV_Q8 ? 1 : 2;
  extern __shared__ __align__(1024) uint8_t smem[];
  // (launched when all before it is done: nothing to wait for)
  const Unit u = unit_of(a);
  const int tile0 = u.rt * PROWS;
  if (idle(a, u, tile0)) {
    pdl_trigger();
    return;
  }
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const uint32_t sb = shaddr(smem);
  // barriers: K and scales ready x 4, V ready x 2; the TMEM address, the abort
  // flag; all products done; for each block of 128 rows: S full x 2, P ready x 2, PV done x 2; Q ready
  const uint32_t bar = sb + L::BAR, kready = bar, vready = bar + 32, done = bar + 56, blocks = bar + 64, qready = bar + 160;
  volatile int *abort = reinterpret_cast<volatile int *>(smem + L::BAR + 52);
  const int nblk = min(2, (u.rows - tile0 + 127) / 128);  // that have rows
  auto sfull_of = [&](int blk, int i) { return blocks + 48 * blk + 8 * (i & 1); };
  auto pready_of = [&](int blk, int i) { return blocks + 48 * blk + 16 + 8 * (i & 1); };
  auto pvdone_of = [&](int blk, int i) { return blocks + 48 * blk + 32 + 8 * (i & 1); };
  if (tid == 0) {
    for (int i = 0; i < 4; i++) mbar_init(kready + 8 * i, 2 * PCONV);  // (each thread after each half of a tile)
    for (int i = 0; i < 2; i++) {
      mbar_init(vready + 8 * i, 2 * PCONV);
      for (int m = 0; m < 2; m++) {
        mbar_init(sfull_of(m, i), 2);  // the products, and the warp that issues them (which has seen the scales)
        mbar_init(pready_of(m, i), 128);
        mbar_init(pvdone_of(m, i), 1);
      }
    }
    mbar_init(done, 1);
    mbar_init(qready, PSOFT);
    *abort = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (warp == PWS + 8) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(bar + 48), "r"(2 * L::COLS) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  pdl_trigger();
  const uint32_t tmem = *reinterpret_cast<volatile uint32_t *>(smem + L::BAR + 48);
  const int hi = u.hi, nt = (hi - u.lo + PK_N - 1) / PK_N;  // (at least one)

  if (warp >= PWS + 8) {  // ------------------------------------------- products
    set_regs<false, PREGS_MMA>();
    if (warp == PWS + 8 && elect_one()) {
      const uint64_t qd = tc_desc(sb + L::Q, PROWS * 16, 128), kd = tc_desc(sb + L::K, L::CH, 128), vd = tc_desc(sb + L::V, 128, L::CH);
      auto scores = [&](int i, int m) {
        const uint64_t q = qd + m * 128, k = kd + (i & 1) * (L::TILE / 16);
#pragma unroll 1
        for (int s = 0; s < DH / 16; s++)
          mma_f16<PK_N, false>(tmem + m * L::COLS + L::S_COL, q + s * 2 * PROWS, k + s * 2 * (L::CH / 16), s > 0);
        mbar_arrive(sfull_of(m, i));
        commit_one(sfull_of(m, i));
      };
      wait_one(qready, 0, abort);
      wait_one(kready, 0, abort);
      tc_fence_after();
      for (int m = 0; m < nblk; m++) scores(0, m);
      for (int i = 0; i < nt; i++) {
        wait_one(vready + 8 * (i & 1), (i >> 1) & 1, abort);
        if (i + 1 < nt) wait_one(kready + 8 * ((i + 1) & 3), ((i + 1) >> 2) & 1, abort);
        for (int m = 0; m < nblk; m++) {
          wait_one(pready_of(m, i), (i >> 1) & 1, abort);
          tc_fence_after();
          const uint32_t w = tmem + m * L::COLS + L::S_COL, o = tmem + m * L::COLS + L::O_COL;
          const uint64_t v = vd + (i & 1) * (L::TILE / 16);
#pragma unroll 1
          for (int s = 0; s < PK_N / 16; s++) mma_f16_ts<DH, true>(o, w + s * 8, v + s * 16, i > 0 || s > 0);
          commit_one(pvdone_of(m, i));
          if (i + 1 < nt) scores(i + 1, m);  // (over the weights just used: products are done in order)
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
  } else if (tid >= PSOFT) {  // --------------------------------------- codes
    // 64 positions at a time, two such halves a tile; who loads what as in
    // pk_cache_attn_tc.cu: 16 bytes of a row a lane (RL lanes a row), NP passes of
    // RP rows, eight lanes that store together touching every bank once.
    set_regs<false, PREGS_CONV>();
    const bool is_v = warp >= PWS + 4;
    constexpr int RL = RB / 16, RP = PCONV / RL, NP = 64 / RP;
    constexpr int RS = TYPE == PK_KV_Q8 ? 4 : 2;
    const int ct = (tid - PSOFT) & (PCONV - 1);
    const int sub = RL <= RS ? ct % RL : ct % RS + (ct / 8 % (RL / RS)) * RS;
    const int key0 = RL <= RS ? ct / RL : ct / RS % (8 / RS) + ct / (8 * RL / RS) * (8 / RS);
    static_assert(RP % 16 == 0, "a pass has whole groups of 16 rows");
    uint4 raw[NP];  // the next half's codes and sub-scales
    uint32_t subs[TYPE == PK_KV_Q4 ? NP : 1];
    float dk = 0.0f, dv = 0.0f;
    bool on = false;
    // Lane x of every warp holds, for the next 8 halves, the cache rows of
    // positions 16 (x & 3) .. of half x >> 2, in units of 16 rows: -1 where there
    // is no page.  Such rows are read from the cache's first.
    int rows16 = -1;
    const uint8_t *codes = reinterpret_cast<const uint8_t *>(is_v ? a.c.v : a.c.k);
    const uint32_t *subs_of = reinterpret_cast<const uint32_t *>(is_v ? a.c.vs : a.c.ks);
    auto ask = [&](int h) {
      if (!(h & 7)) {
        const int p = u.lo + 64 * (h + (lane >> 2)) + 16 * (lane & 3), j = p >> a.page_shift;
        const int pg = p < hi && j < a.s.max_pages ? __ldg(a.s.pages + (size_t)u.s * a.s.max_pages + j) : -1;
        rows16 = pg >= 0 && pg < a.c.n_pages
                     ? (int)((((long long)pg * a.c.n_kv + u.h) * a.c.page_size + (p & (a.c.page_size - 1))) >> 4)
                     : -1;
      }
#pragma unroll
      for (int w = 0; w < NP; w++) {
        const uint32_t r = max(__shfl_sync(0xffffffffu, rows16, 4 * (h & 7) + w * (RP / 16) + key0 / 16), 0);
        raw[w] = __ldcg(reinterpret_cast<const uint4 *>(codes + ((size_t)r * (16 * RB) + ((key0 & 15) * RB + 16 * sub))));
        if (TYPE == PK_KV_Q4) subs[w] = __ldcg(subs_of + ((size_t)r * (16 * SW) + ((key0 & 15) * SW + 1)));
      }
      if (!is_v && !(h & 1)) {  // the tile's scales, a position a thread
        const int r = __shfl_sync(0xffffffffu, rows16, 4 * (h & 7) + ct / 16);
        on = r >= 0 && u.lo + 64 * h + ct < hi;
        const size_t at = (size_t)max(r, 0) * (16 * SW) + (ct & 15) * SW;
        dk = __ldcg(a.c.ks + at);
        dv = __ldcg(a.c.vs + at);
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
    // in place of tile i - 4's: K's buffer is free, so tile i - 2's scores are
    // there and tile i - 4's weights have been used
    auto put_scales = [&](int i) {
      uint8_t *sc = smem + L::SC + (i & 3) * L::SCB;
      float *f = reinterpret_cast<float *>(sc);
      f[ct] = on ? fminf(fmaxf(dk * (a.q.scale * kLog2e), -3e38f), 3e38f) : 0.0f;  // (finite: a query may be 0)
      f[PK_N + ct] = on ? dv : 0.0f;
      f[2 * PK_N + ct] = on ? 0.0f : -CUDART_INF_F;
      f[3 * PK_N + ct] = on ? log2f(fabsf(dv)) : -CUDART_INF_F;
      const unsigned m = __ballot_sync(0xffffffffu, on);
      const uint32_t x = __reduce_max_sync(0xffffffffu, on ? __float_as_uint(dv) & 0x7fffffffu : 0);
      if (lane == 0) {
        reinterpret_cast<uint32_t *>(sc + 4 * PK_N * 4)[ct >> 5] = m;
        reinterpret_cast<uint32_t *>(sc + 4 * PK_N * 4 + 16)[ct >> 5] = x;
      }
    };
    const int n = 2 * nt;
    ask(0);
    for (int h = 0; h < n; h++) {
      const int i = h >> 1;
      // K's buffer is free once tile i - 2's scores are there, V's once its
      // products with V are
      if (i >= 2 && !(h & 1))
        for (int m = 0; m < nblk; m++) wait(is_v ? pvdone_of(m, i) : sfull_of(m, i), ((i - 2) >> 1) & 1, abort);
      put(sb + (is_v ? L::V : L::K) + (i & 1) * L::TILE + (h & 1) * 64 * 16);
      if (!is_v && !(h & 1)) put_scales(i);
      fence_async_smem();
      mbar_arrive(is_v ? vready + 8 * (i & 1) : kready + 8 * (i & 3));
      if (h + 1 < n) ask(h + 1);
    }
  } else {  // ------------------------------------------------------------ softmax
    set_regs<true, PREGS_SOFT>();
    const int blk = warp >> 2;
    const uint32_t lanes = ((uint32_t)((warp & 3) * 32) << 16) + blk * L::COLS;
    const bool work = tile0 + warp * 32 < u.rows;  // (the whole warp)
    const int row = tile0 + tid, quad = lane & 3;
    const uint32_t cols = tmem + lanes + L::S_COL;
    // of rows lane / 4 + 8 j: the scale, the reference, this thread's part of the sum
    // (the scale and less the reference as pairs, too)
    float rs4[4] = {1.0f, 1.0f, 1.0f, 1.0f}, m4[4], l4[4];
    put_q_rows<TYPE, DH, E>(a, u, tile0 + warp * 32, sb + L::Q + warp * 32 * 16, rs4);
    fence_async_smem();
    mbar_arrive(qready);
    uint64_t scale2[4], less4[4];
#pragma unroll
    for (int j = 0; j < 4; j++) {
      scale2[j] = pair_of(rs4[j], rs4[j]);
      less4[j] = 0;
      m4[j] = -CUDART_INF_F;
      l4[j] = 0.0f;
    }
    auto pv_wait = [&](int i) { wait(pvdone_of(blk, i), (i >> 1) & 1, abort); };
    if (blk < nblk)
      for (int i = 0; i < nt; i++) {
        wait(sfull_of(blk, i), (i >> 1) & 1, abort);
        tc_fence_after();
        if (work) {
          const uint8_t *sc = smem + L::SC + (i & 3) * L::SCB;
          const uint64_t *dk2 = reinterpret_cast<const uint64_t *>(sc) + quad, *dv2 = dk2 + PK_N / 2, *off2 = dk2 + PK_N, *log2v = dk2 + 3 * (PK_N / 2);
          const uint4 held = *reinterpret_cast<const uint4 *>(sc + 4 * PK_N * 4), r4 = *reinterpret_cast<const uint4 *>(sc + 4 * PK_N * 4 + 16);
          const float vmax = fmaxf(fmaxf(__uint_as_float(r4.x), __uint_as_float(r4.y)), fmaxf(__uint_as_float(r4.z), __uint_as_float(r4.w)));
          const bool masked = (held.x & held.y & held.z & held.w) != 0xffffffffu;
          uint32_t w[2][32];
          uint64_t sum[4];
          // the weights of the products in t, columns 16 k .. of 128, less the references
          auto weights = [&](int k, const float (&t)[16], const uint64_t (&less)[4], bool add) {
#pragma unroll
            for (int g = 0; g < 2; g++) {
              const uint64_t dk = dk2[4 * (2 * k + g)], dv = dv2[4 * (2 * k + g)], off = add ? off2[4 * (2 * k + g)] : 0;
#pragma unroll
              for (int j = 0; j < 4; j++) {
                const int p = 4 * (j >> 1) + 2 * g + (j & 1), at = 2 * (2 * k + g) + (j & 1);
                uint64_t x = pair_of(t[2 * p], t[2 * p + 1]);
                x = F16 ? fma2(x, dk, less[j]) : fma2(mul2(x, dk), scale2[j], less[j]);
                if (add) x = add2(x, off);
                float2 y = unpair(x);
                y.x = ex2(y.x);
                y.y = ex2(y.y);
                x = pair_of(y.x, y.y);
                sum[j] = add2(sum[j], x);
                y = unpair(mul2(x, dv));
                w[j >> 1][at] = pack2(y.x, y.y);
              }
            }
          };
          auto all_weights = [&](const uint64_t (&less)[4], bool add) {
            sum[0] = sum[1] = sum[2] = sum[3] = 0;
            __syncwarp();
            float t[2][16];  // 16 columns are on their way while those before are worked on
            ask_quads(cols, t[0]);
#pragma unroll
            for (int k = 0; k < 8; k++) {
              wait16(t[k & 1]);
              if (k < 7) ask_quads(cols + 16 * (k + 1), t[(k + 1) & 1]);
              weights(k, t[k & 1], less, add);
            }
          };
          bool longer = masked || i == 0;  // (the first tile has no reference yet)
          if (!longer) {
            all_weights(less4, false);
            // (a thread's part of a row's sum is at least the largest of its weights)
            bool over = false;
#pragma unroll
            for (int j = 0; j < 4; j++) {
              const float2 y = unpair(sum[j]);
              const float all = y.x + y.y;
              over |= !(all * vmax <= TOP && all <= 0x1p100f);
            }
            longer = __any_sync(0xffffffffu, over);
          }
          if (longer) {
            float mx[4], top[4], f[4];
#pragma unroll
            for (int j = 0; j < 4; j++) mx[j] = top[j] = -CUDART_INF_F;
            auto quad_max = [](float x) {
              x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 1));
              return fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 2));
            };
            // (of a tile with nothing in it mx is -inf, and its products NaN, which count for nothing)
#pragma unroll 1
            for (int k = 0; k < 8; k++) {
              float t[16];
              __syncwarp();
              ask_quads(cols + 16 * k, t);
              wait16(t);
#pragma unroll
              for (int g = 0; g < 2; g++) {
                const float2 dk = unpair(dk2[4 * (2 * k + g)]), lv = unpair(log2v[4 * (2 * k + g)]), off = unpair(off2[4 * (2 * k + g)]);
#pragma unroll
                for (int j = 0; j < 4; j++) {
                  const int p = 4 * (j >> 1) + 2 * g + (j & 1);
                  const float x = fmaf(t[2 * p] * dk.x, rs4[j], off.x), y = fmaf(t[2 * p + 1] * dk.y, rs4[j], off.y);
                  mx[j] = fmaxf(mx[j], fmaxf(x, y));
                  top[j] = fmaxf(top[j], fmaxf(x + lv.x, y + lv.y));
                }
              }
            }
            bool moved = false;
            uint64_t now4[4];
#pragma unroll
            for (int j = 0; j < 4; j++) {
              f[j] = 1.0f;
              mx[j] = quad_max(mx[j]);
              const float most = fmaxf(quad_max(top[j]), mx[j] - 100.0f);  // the largest product's exponent
              if (mx[j] != -CUDART_INF_F && (m4[j] == -CUDART_INF_F || most > m4[j] + 8.0f || mx[j] > m4[j] + 90.0f)) {
                const float now = fmaxf(most - 6.0f, mx[j] - 90.0f);
                f[j] = ex2(m4[j] - now);
                l4[j] *= f[j];
                m4[j] = now;
                moved |= f[j] != 1.0f;
              }
              // (nothing seen yet: all are masked; the next tile's weights will be infinite)
              less4[j] = pair_of(-m4[j], -m4[j]);
              now4[j] = m4[j] == -CUDART_INF_F ? 0 : less4[j];
            }
            if (i > 0 && __any_sync(0xffffffffu, moved)) {  // O's rows, once the products before are done
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
            all_weights(now4, true);
          }
#pragma unroll
          for (int j = 0; j < 4; j++) {
            const float2 y = unpair(sum[j]);
            l4[j] += y.x + y.y;
          }
          __syncwarp();
          // the weights take their scores' columns, two a column
#pragma unroll
          for (int q = 0; q < 4; q++) st_pairs(cols + 16 * q, w[0] + 8 * q, w[1] + 8 * q);
          asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory");
        }
        tc_fence_before();
        mbar_arrive(pready_of(blk, i));
      }
    // ---- the rows, by way of the operands' place: all blocks' products are done
    if (blk < nblk) pv_wait(nt - 1);
    tc_fence_after();
    float m = 0.0f, l = 0.0f;  // one row a lane again
#pragma unroll
    for (int j = 0; j < 4; j++) {
      float x = l4[j];
      x += __shfl_xor_sync(0xffffffffu, x, 1);
      x += __shfl_xor_sync(0xffffffffu, x, 2);
      x = __shfl_sync(0xffffffffu, x, 4 * (lane & 7));
      const float y = __shfl_sync(0xffffffffu, m4[j], 4 * (lane & 7));
      if ((lane >> 3) == j) l = x, m = y;
    }
    asm volatile("bar.sync 1, %0;" ::"r"(PSOFT) : "memory");
    if (work) {
      const bool on = row < u.rows;
      const int r = min(row, u.rows - 1), i = r / a.group, h = u.h * a.group + r - i * a.group;
      const long long slot = ((long long)(u.sv.first + i) * a.q.n_head + h) * a.n_part + u.slot;
      const float f = *abort ? CUDART_NAN_F : l == 0.0f ? 0.0f : 1.0f;
      if (on) a.part_ml[slot] = make_float2(m, *abort ? CUDART_NAN_F : l);
      float *so = reinterpret_cast<float *>(smem) + tid * (DH + 4);
#pragma unroll 1
      for (int c = 0; c < DH / 16; c++) {
        float v[16];
        __syncwarp();
        ld16(tmem + lanes + L::O_COL + 16 * c, v);
#pragma unroll
        for (int k = 0; k < 2; k++) {
          float x[8];
#pragma unroll
          for (int j = 0; j < 8; j++) x[dim8<TYPE>(j)] = f == 0.0f ? 0.0f : v[8 * k + j] * f;
          store_n<float, 8>(so + 16 * c + 8 * k, true, x);
        }
      }
      __syncwarp();
      constexpr int LR = DH / 4, RP = 32 / LR;  // lanes a row, rows at a time
      const int sub = lane / LR, d0 = (lane % LR) * 4, rows = min(32, u.rows - tile0 - warp * 32);
#pragma unroll 4
      for (int r0 = 0; r0 < rows; r0 += RP) {
        const int x = min(r0 + sub, 31);
        const long long to = __shfl_sync(0xffffffffu, slot, x) * DH + d0;
        const float4 v = *reinterpret_cast<const float4 *>(reinterpret_cast<const float *>(smem) + (warp * 32 + x) * (DH + 4) + d0);
        if (r0 + sub < rows) *reinterpret_cast<float4 *>(a.part_o + to) = v;
      }
    }
    __syncwarp();
    set_regs<false, PREGS>();
  }
  tc_fence_before();
  __syncthreads();
  // Only here, after the softmax warps have had their registers and given them
  // back: taken earlier they would be missing there.
  if (warp >= PWS) set_regs<true, PREGS>();
  if (warp == PWS + 8) {
    tc_fence_after();
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(2 * L::COLS) : "memory");
  }
}

template <class E>
void (*prefix_kernel(const pk_kv_cache &c, int &smem))(AttnKArgs) {
  smem = c.head_dim == 64 ? PLay<64>::BYTES : PLay<128>::BYTES;
  if (c.head_dim == 64) return c.type == PK_KV_Q8 ? k_kv_prefix<PK_KV_Q8, 64, E> : k_kv_prefix<PK_KV_Q4, 64, E>;
  return c.type == PK_KV_Q8 ? k_kv_prefix<PK_KV_Q8, 128, E> : k_kv_prefix<PK_KV_Q4, 128, E>;
}

}  // namespace

cudaError_t launch_kv_prefix(const AttnKArgs &a, unsigned blocks, cudaStream_t st) {
  int smem = 0;
  const bool f16 = a.q.type == T_F16;
  const auto k = f16 ? prefix_kernel<__half>(a.c, smem) : prefix_kernel<__nv_bfloat16>(a.c, smem);
  // the split of the registers would wait forever for what a launch does not have
  static std::atomic<unsigned> checked{0};
  const unsigned bit = 1u << (4 * f16 + 2 * (a.c.type == PK_KV_Q4) + (a.c.head_dim == 128));
  if (!(checked.load(std::memory_order_relaxed) & bit)) {
    cudaFuncAttributes f;
    const cudaError_t err = cudaFuncGetAttributes(&f, reinterpret_cast<const void *>(k));
    if (err != cudaSuccess) return err;
    if (f.numRegs != PREGS) return cudaErrorInvalidConfiguration;
    checked.fetch_or(bit, std::memory_order_relaxed);
  }
  return launch_as(false, k, 1, dim3(blocks), dim3(PTHREADS), smem, st, a);
}

}  // namespace pk
