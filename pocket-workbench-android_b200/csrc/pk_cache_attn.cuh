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
  float *part_o;   // [n_tok][n_head][n_chunk][DH]: chunks' parts, or what long sums gave up so far
  float2 *part_ml; // [n_tok][n_head][n_chunk]
  int chunk, n_chunk, row_tiles, group, page_shift, vec_q, vec_o;
  int cluster;  // 1: a sequence's chunks are a cluster's CTAs, which add up among themselves
  int *err;     // null, or a device word that PK_ERR_TIMEOUT goes to when a bounded wait ran out
  int poison;   // 1 (self-test): the codes never arrive, so that the waits run out
};

// A CTA's work: one chunk of positions [lo, hi) for one tile of the rows (token
// i, query head of kv head h) of one sequence.  Sequences of more than one
// chunk (nch) leave theirs in the scratch, or to the cluster.
struct Unit {
  SeqView sv;
  int s, h, rt, ch, lo, hi, nch, rows;
};
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
  u.sv = seq_view(a.s, a.c.page_size, u.s);
  u.rows = u.sv.n * a.group;
  u.nch = (u.sv.total + a.chunk - 1) / a.chunk;
  u.lo = u.ch * a.chunk;
  u.hi = min(u.sv.total, u.lo + a.chunk);
  return u;
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
    float *p = a.part_o + ((tok * a.q.n_head + h) * a.n_chunk + u.ch) * DH + d0;
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
// rows of a kv head a CTA (two CTAs an SM, or one).
cudaError_t launch_kv_attn_tc(const AttnKArgs &a, int cluster, unsigned blocks, cudaStream_t st);

}  // namespace pk
