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

__device__ __forceinline__ void cp16(uint32_t dst, const void *src) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
}
__device__ __forceinline__ void cp_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void cp_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }

struct AttnKArgs {
  pk_kv_cache c;
  pk_kv_seqs s;
  pk_kv_query q;
  float *part_o;   // [n_tok][n_head][n_chunk][DH]
  float2 *part_ml; // [n_tok][n_head][n_chunk]
  int chunk, n_chunk, row_tiles, group, page_shift, vec_q, vec_o;
};

// A CTA's work: one chunk of positions [lo, hi) for one tile of the rows (token
// i, query head of kv head h) of one sequence.  Sequences of more than one
// chunk (nch) leave theirs in the scratch.
struct Unit {
  SeqView sv;
  int s, h, rt, ch, lo, hi, nch, rows;
};
__device__ __forceinline__ Unit unit_of(const AttnKArgs &a) {
  Unit u;
  unsigned id = blockIdx.x;
  u.rt = (int)(id % (unsigned)a.row_tiles);
  id /= (unsigned)a.row_tiles;
  u.h = (int)(id % (unsigned)a.c.n_kv);
  id /= (unsigned)a.c.n_kv;
  u.ch = (int)(id % (unsigned)a.n_chunk);
  u.s = (int)(id / (unsigned)a.n_chunk);
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


// The tcgen05 kernel's launch (pk_cache_attn_tc.cu): 128 rows of a kv head's
// tile, half-precision queries.
constexpr int TC_ATTN_ROWS = 128;
cudaError_t launch_kv_attn_tc(const AttnKArgs &a, unsigned blocks, cudaStream_t st);

}  // namespace pk
