// pk_cache_attn.cuh -- what the two kernels of the attention over the
// quantised cache share (pk_cache_attn.cu, pk_cache_attn_tc.cu).
#pragma once
#include <math_constants.h>

#include "pk_cache.cuh"
#include "pk_cache.h"

namespace pk {

constexpr float kLog2e = 1.4426950408889634f;
// M moves when the maximum passes it by 2^GROW; a row's factor inv is set so
// that its largest weight times scale is SET and set again past TOP (f16 ends
// at 65504), so what rounds to a subnormal is below 2^-20 of the largest.
constexpr float GROW = 6.0f, SET = 64.0f, TOP = 32768.0f;

__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
// (a, b) as two f16 and, for the second term, what the rounding left.
__device__ __forceinline__ uint32_t pack2(float a, float b) { return h2u(__floats2half2_rn(a, b)); }
__device__ __forceinline__ uint32_t rest2(float a, float b, uint32_t hi) {
  const float2 f = __half22float2(u2h(hi));
  return pack2(a - f.x, b - f.y);
}

// x, and NaN for infinities: a query's infinity would give scores of -inf where
// all codes that it meets have the other sign, as if nothing were seen.
__device__ __forceinline__ float inf_nan(float x) { return x + (x - x); }

__device__ __forceinline__ void cp16(uint32_t dst, const void *src) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
}
__device__ __forceinline__ void cp_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void cp_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }

// Half-precision queries' outputs are summed by the tensor core, which cuts off
// what it shifts out: less than 2^-23 of the sum each step of 16 positions, all
// to one side where V's values have one sign (measured: 2^-27.1 of it a position
// on tcgen05, a quarter on mma.sync, whose four groups of warps have sums of
// their own).  A sum goes over so many positions that this stays under an eighth
// of the output's rounding, 2^-14 for f16 and 2^-11 for bf16; then on mma.sync
// the chunk ends, and on tcgen05 the sum is added to the scratch in f32.
__host__ __device__ constexpr int sum_most(int type) { return type == T_F16 ? 8192 : 65536; }

struct AttnKArgs {
  pk_kv_cache c;
  pk_kv_seqs s;
  pk_kv_query q;
  float *part_o;   // [n_tok][n_head][n_part][DH]: chunks' parts, or what long sums gave up so far
  float2 *part_ml; // [n_tok][n_head][n_part]
  int chunk, n_chunk, row_tiles, group, page_shift, vec_q, vec_o;
  int cluster;  // 1: a sequence's chunks are a cluster's CTAs, which add up among themselves
  int *err;     // null, or a device word that PK_ERR_TIMEOUT goes to when a bounded wait ran out
  int poison;   // 1 (self-test): the codes never arrive, so that the waits run out
  // What a launch goes over: all of each sequence, each group's shared prefix,
  // or what each sequence has besides it.  The last two leave their chunks'
  // parts in the scratch, a row's n_part of them: the prefix's from 0 on, its
  // own from n_pre on.  merge: what a sequence has besides is one chunk, whose CTA
  // adds the prefix's parts (up to MERGE of them) to its rows and writes them out.
  int mode, part0, n_part, n_pre, pre_chunk, merge;
  // 1: the launch before this one is the prefixes', which began when all earlier
  // work was done, and is waited for only where its parts are needed.
  int early;
  pk_kv_shared sh;
};
constexpr int MERGE = 8;
enum : int { ATTN_ALL = 0, ATTN_PREFIX = 1, ATTN_OWN = 2 };

// Group g's sequences [s0, s1), their tokens [t0, t0 + n), and the positions
// that they share, of which `base`, a multiple of 16 as tiles are, are computed
// for all; none (0) where the group has no tokens, or more than max_tok.
struct GroupView {
  int s0, s1, t0, n, len, base;
};
__device__ __forceinline__ GroupView group_view(const AttnKArgs &a, int g) {
  GroupView v;
  v.s0 = min(max(__ldg(a.sh.first + g), 0), a.s.n_seq);
  v.s1 = min(max(__ldg(a.sh.first + g + 1), v.s0), a.s.n_seq);
  v.t0 = min(max(__ldg(a.s.start + v.s0), 0), a.s.n_tok);
  v.n = min(max(__ldg(a.s.start + v.s1), v.t0), a.s.n_tok) - v.t0;
  const long long cap = min(min((long long)a.s.max_pages * a.c.page_size, (long long)a.s.max_len), (long long)a.sh.max_len);
  v.len = (int)min((long long)max(__ldg(a.sh.len + g), 0), cap);
  if (v.n < 1 || v.n > a.sh.max_tok) v.n = v.len = 0;
  v.base = v.len & ~15;
  return v;
}
// The positions of sequence s (a whole warp asks) that are left to itself: from
// base, which its group's prefix reaches to, up to total.
struct OwnView {
  int base, total;
};
__device__ __forceinline__ OwnView own_view(const AttnKArgs &a, int s, const SeqView &sv) {
  int base = 0, len = 0;
  const int g = a.sh.n_group > 1 ? last_at(a.sh.first, a.sh.n_group, s, threadIdx.x & 31) : a.sh.n_group - 1;
  if (g >= 0) {
    const GroupView v = group_view(a, g);
    if (s >= v.s0 && s < v.s1 && sv.ctx >= v.len) base = v.base, len = v.len;
  }
  return {base, max(base, (int)min((long long)sv.total, (long long)len + a.sh.max_own))};
}

// A CTA's work: one chunk of positions [lo, hi) for one tile of the rows (token
// i, query head of kv head h) of one sequence.  Sequences of more than one
// chunk (nch) leave theirs in the scratch, or to the cluster.
struct Unit {
  SeqView sv;
  int s, h, rt, ch, lo, hi, nch, rows, slot;  // (slot: of its part among a row's)
  bool part;
};
// SHARED: a launch may be a prefix's or what is besides one (a.mode).
template <bool SHARED = true>
__device__ __forceinline__ Unit unit_of(const AttnKArgs &a) {
  Unit u;
  unsigned id = blockIdx.x;
  // a sequence's chunks side by side (a cluster's have to be)
  u.ch = (int)(id % (unsigned)a.n_chunk);
  id /= (unsigned)a.n_chunk;
  u.rt = (int)(id % (unsigned)a.row_tiles);
  id /= (unsigned)a.row_tiles;
  u.h = (int)(id % (unsigned)a.c.n_kv);
  u.s = (int)(id / (unsigned)a.c.n_kv);
  int base = 0;
  if (SHARED && a.mode == ATTN_PREFIX) {
    const GroupView g = group_view(a, u.s);
    u.s = g.s0;  // (whose pages are read)
    u.sv = SeqView{g.t0, g.n, g.base, g.base};
  } else {
    u.sv = seq_view(a.s, a.c.page_size, u.s);
    if (SHARED && a.mode == ATTN_OWN && u.sv.n > 0) {
      const OwnView v = own_view(a, u.s, u.sv);
      base = v.base;
      u.sv.total = v.total;
    }
  }
  u.rows = u.sv.n * a.group;
  u.nch = (u.sv.total - base + a.chunk - 1) / a.chunk;
  u.lo = base + u.ch * a.chunk;
  u.hi = min(u.sv.total, u.lo + a.chunk);
  u.slot = (SHARED ? a.part0 : 0) + u.ch;
  u.part = (SHARED && a.mode != ATTN_ALL && !a.merge) || u.nch > 1;
  return u;
}
// Has this CTA nothing to do?  (Rows that see nothing are written by their first chunk, or by the joining launch.)
template <bool SHARED = true>
__device__ __forceinline__ bool idle(const AttnKArgs &a, const Unit &u, int tile0) {
  if (tile0 >= u.rows) return true;
  return u.ch >= (!SHARED || a.mode == ATTN_ALL || a.merge ? max(u.nch, 1) : u.nch) && !(a.cluster && u.nch > 1);
}
// Beside the prefixes' launch: it is not over before one CTA (the last) has seen
// that end, as what follows waits for this launch alone.
__device__ __forceinline__ void end_early(const AttnKArgs &a) {
  if (a.early && blockIdx.x == gridDim.x - 1) pdl_wait();
}

// A row's sum L of weights 2^(s - M) and the parts of its prefix: the factors by
// which both are added up, f[c] of the parts and `own`, over their common sum.
// (Read past L1, written by a launch that may have run beside this one.)
struct Merge {
  float f[MERGE], own;
  const float *part;
  int n;
};
template <int DH>
__device__ __forceinline__ Merge merge_of(const AttnKArgs &a, const Unit &u, int row, float M, float L) {
  Merge g;
  const int i = row / a.group, h = u.h * a.group + row - i * a.group;
  const long long at = ((long long)(u.sv.first + i) * a.q.n_head + h) * a.n_part;
  g.n = (u.lo + a.pre_chunk - 1) / a.pre_chunk;  // (one chunk: it begins where the prefix ends)
  g.part = a.part_o + at * DH;
  float2 ml[MERGE];
  float top = L == 0.0f ? -CUDART_INF_F : M;
#pragma unroll
  for (int c = 0; c < MERGE; c++) {
    ml[c] = c < g.n ? __ldcg(a.part_ml + at + c) : make_float2(-CUDART_INF_F, 0.0f);
    top = fmaxf(top, ml[c].x);
  }
  g.own = L == 0.0f ? 0.0f : ex2(M - top);  // a NaN sum stays one
  float all = g.own * L;
#pragma unroll
  for (int c = 0; c < MERGE; c++) {
    g.f[c] = ml[c].y == 0.0f ? 0.0f : ex2(ml[c].x - top);
    all = fmaf(g.f[c], ml[c].y, all);
  }
  const float inv = all > 0.0f || isnan(all) ? 1.0f / all : 0.0f;
  g.own *= inv;
#pragma unroll
  for (int c = 0; c < MERGE; c++) g.f[c] *= inv;
  return g;
}
// N elements from d0 on.  (All parts' loads of four elements are asked for together.)
template <int N>
__device__ __forceinline__ void merge_in(const Merge &g, int dh, int d0, float (&x)[N]) {
#pragma unroll
  for (int j = 0; j < N; j++) x[j] = g.own == 0.0f ? 0.0f : x[j] * g.own;
  const float4 *p = reinterpret_cast<const float4 *>(g.part + d0);
#pragma unroll
  for (int j = 0; j < N / 4; j++) {
    float4 v[MERGE];
#pragma unroll
    for (int c = 0; c < MERGE; c++) {
      v[c] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
      if (c < g.n) v[c] = __ldcg(p + j + (size_t)c * (dh / 4));
    }
#pragma unroll
    for (int c = 0; c < MERGE; c++) {
      if (c < g.n && g.f[c] != 0.0f) {
        x[4 * j] = fmaf(g.f[c], v[c].x, x[4 * j]);
        x[4 * j + 1] = fmaf(g.f[c], v[c].y, x[4 * j + 1]);
        x[4 * j + 2] = fmaf(g.f[c], v[c].z, x[4 * j + 2]);
        x[4 * j + 3] = fmaf(g.f[c], v[c].w, x[4 * j + 3]);
      }
    }
  }
}

// Does row (token i) see draft j?
__device__ __forceinline__ bool sees(const AttnKArgs &a, const Unit &u, int i, int j) {
  if (j >= u.sv.n) return false;
  if (!a.q.mask) return j <= i;
  if ((j >> 6) >= a.q.mask_words) return false;
  return (__ldg(a.q.mask + (size_t)(u.sv.first + i) * a.q.mask_words + (j >> 6)) >> (j & 63)) & 1;
}


// Every thread of the cluster arrives, and sees what the others wrote before.
__device__ __forceinline__ void cluster_sync() {
  asm volatile("barrier.cluster.arrive.release.aligned;\n barrier.cluster.wait.acquire.aligned;" ::: "memory");
}
__device__ __forceinline__ uint32_t at_rank(uint32_t addr, int rank) {
  uint32_t r;
  asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(addr), "r"(rank));
  return r;
}
__device__ __forceinline__ float4 ld_cluster4(uint32_t a) {
  float4 v;
  asm volatile("ld.shared::cluster.v4.f32 {%0,%1,%2,%3}, [%4];" : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w) : "r"(a) : "memory");
  return v;
}
__device__ __forceinline__ float2 ld_cluster2(uint32_t a) {
  float2 v;
  asm volatile("ld.shared::cluster.v2.f32 {%0,%1}, [%2];" : "=f"(v.x), "=f"(v.y) : "r"(a) : "memory");
  return v;
}

// Writes DH / 8 elements of a row: final (out), or the chunk's part.
template <int DH>
__device__ __forceinline__ void write_row(const AttnKArgs &a, const Unit &u, int row, int d0, const float (&x)[DH / 8], bool part) {
  const int i = row / a.group, h = u.h * a.group + row - i * a.group;
  const long long tok = u.sv.first + i;
  if (part) {
    float *p = a.part_o + ((tok * a.q.n_head + h) * a.n_part + u.slot) * DH + d0;
#pragma unroll
    for (int j = 0; j < DH / 8; j += 4) *reinterpret_cast<float4 *>(p + j) = make_float4(x[j], x[j + 1], x[j + 2], x[j + 3]);
    return;
  }
  const long long off = tok * a.q.out_tok_stride + (long long)h * a.q.out_head_stride + d0;
  if (a.q.type == T_F32) store_n<float, DH / 8>(reinterpret_cast<float *>(a.q.out) + off, a.vec_o, x);
  else if (a.q.type == T_F16) store_n<__half, DH / 8>(reinterpret_cast<__half *>(a.q.out) + off, a.vec_o, x);
  else store_n<__nv_bfloat16, DH / 8>(reinterpret_cast<__nv_bfloat16 *>(a.q.out) + off, a.vec_o, x);
}

// The rows of a cluster's chunks added up: each CTA has its rows' sums at
// shared address so ([row][DH + 4] f32) and their (M, L) at sml, and takes
// every nch-th group of DH / 8 elements.  All threads of all CTAs call it
// after the sums are written; a CTA without a chunk only keeps step.
template <int DH>
__device__ __forceinline__ void join_cluster(const AttnKArgs &a, const Unit &u, int tile0, int rows, uint32_t so, uint32_t sml, int threads) {
  cluster_sync();
  if (u.ch < u.nch) {
    for (int x = u.ch * threads + (int)threadIdx.x; x < rows * 8; x += u.nch * threads) {
      const int r = x >> 3, d0 = (x & 7) * (DH / 8);
      if (tile0 + r >= u.rows) continue;
      float2 ml[8];
      float M = -CUDART_INF_F, L = 0.0f, acc[DH / 8];
#pragma unroll
      for (int c = 0; c < 8; c++) {
        ml[c] = make_float2(-CUDART_INF_F, 0.0f);
        if (c < u.nch) ml[c] = ld_cluster2(at_rank(sml + r * 8, c));
        M = fmaxf(M, ml[c].x);
      }
#pragma unroll
      for (int j = 0; j < DH / 8; j++) acc[j] = 0.0f;
#pragma unroll
      for (int c = 0; c < 8; c++) {
        if (c >= u.nch) continue;
        const float f = ml[c].y == 0.0f ? 0.0f : ex2(ml[c].x - M);  // a NaN sum stays one
        L = fmaf(f, ml[c].y, L);
        const uint32_t p = at_rank(so + (r * (DH + 4) + d0) * 4, c);
#pragma unroll
        for (int j = 0; j < DH / 8; j += 4) {
          const float4 v = ld_cluster4(p + 4 * j);
          acc[j] = fmaf(f, v.x, acc[j]);
          acc[j + 1] = fmaf(f, v.y, acc[j + 1]);
          acc[j + 2] = fmaf(f, v.z, acc[j + 2]);
          acc[j + 3] = fmaf(f, v.w, acc[j + 3]);
        }
      }
      const float inv = L > 0.0f || isnan(L) ? 1.0f / L : 0.0f;
#pragma unroll
      for (int j = 0; j < DH / 8; j++) acc[j] *= inv;
      write_row<DH>(a, u, tile0 + r, d0, acc, false);
    }
  }
  cluster_sync();  // (until then the others may be reading)
}

// The tcgen05 kernel's launch (pk_cache_attn_tc.cu): one or two blocks of 128
// rows of a kv head a CTA (two CTAs an SM, or one; two for f32 alone).
cudaError_t launch_kv_attn_tc(const AttnKArgs &a, int rows, int cluster, unsigned blocks, cudaStream_t st);
// The shared prefixes' of many half-precision rows, 256 a CTA (pk_cache_prefix.cu).
constexpr int PREFIX_ROWS = 256;
cudaError_t launch_kv_prefix(const AttnKArgs &a, unsigned blocks, cudaStream_t st);

}  // namespace pk
