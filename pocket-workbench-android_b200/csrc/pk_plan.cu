// pk_plan.cu -- page tables and slot maps of a step from the requests' lengths
// (pk_kv_plan).  No counterpart in the reference, whose cache is one sequence's
// array (model.rs:352-387).
//
// With n_s the tokens of slot s, cut so that their sum is at most n_tok, P the
// page size and h_s the pages held:
//   start_s = sum of n before s        (sums that stop at n_tok: min(a + b, n_tok)
//                                       is associative, so they can be scanned)
//   take_s  = max(0, min(max_pages, ceil((ctx_s + n_s) / P)) - h_s), n_s > 0
//   back_s  = h_s - shared_s of done slots
// Entry i of the list is free[i], or a page given back; the page taken k-th is
// entry n_free + sum(back) - 1 - k.  So a page, a token's slot and an entry of
// the new list each follow from the three prefix sums alone, and every CTA makes
// them for itself in shared memory (one pass over 12 bytes a slot from L2) and
// then takes its share of the tokens, of the taken pages, of the list and, with
// new tables, of their rows: one launch, no CTA waits for another.  In place
// what is read is also written: there a cluster of 8 CTAs does all of it, and
// what others may still read (counts, entries that become -1) is written
// behind the cluster's barrier.
//
// Measured: 24 slots of 256 pages, a token each: 6 us; 1000 slots of 1024 pages,
// an eighth of them done, an eighth with prompts (34,000 tokens), new tables of
// 4 MB: 12 us, twice what the bytes take.  What bounds it: the loads that depend
// on one another (lengths, then counts, then the list's entries); a call from
// Python takes 20 us.
#include <algorithm>

#include "pk_cache.cuh"
#include "pk_cache.h"
#include "pk_launch.h"

namespace pk {
namespace {

constexpr int PT = 512;  // threads
constexpr int PW = PT / 32;

// Exclusive prefix sums over a CTA of up to two numbers a thread, min(a + b, cap) each; the sums of all into total.
struct Pair {
  uint32_t a, b;
};
__device__ __forceinline__ uint32_t add_to(uint32_t x, uint32_t y, uint32_t cap) { return min(x + y, cap); }
__device__ __forceinline__ Pair scan2(Pair v, uint32_t cap, Pair *sums, Pair &total) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  Pair x = v;
#pragma unroll
  for (int i = 1; i < 32; i *= 2) {
    const uint32_t a = __shfl_up_sync(0xffffffffu, x.a, i), b = __shfl_up_sync(0xffffffffu, x.b, i);
    if (lane >= i) x.a = add_to(x.a, a, cap), x.b = add_to(x.b, b, cap);
  }
  if (lane == 31) sums[warp] = x;
  __syncthreads();
  Pair before{0, 0};
  total = before;
#pragma unroll
  for (int w = 0; w < PW; w++) {
    const Pair s = sums[w];
    if (w < warp) before.a = add_to(before.a, s.a, cap), before.b = add_to(before.b, s.b, cap);
    total.a = add_to(total.a, s.a, cap), total.b = add_to(total.b, s.b, cap);
  }
  // (exclusive: the sum of the lanes before)
  uint32_t a = __shfl_up_sync(0xffffffffu, x.a, 1), b = __shfl_up_sync(0xffffffffu, x.b, 1);
  if (lane == 0) a = b = 0;
  __syncthreads();  // sums may be written again
  return {add_to(before.a, a, cap), add_to(before.b, b, cap)};
}

// The last i < n with at[i] <= x (at[0] <= x).
__device__ __forceinline__ int last_at(const uint32_t *at, int n, uint32_t x) {
  int lo = 0;
  while (n > 1) {
    const int half = n >> 1;
    if (at[lo + half] <= x) lo += half;
    n -= half;
  }
  return lo;
}

// What may also be written, in place, is read as such.
template <bool IN_PLACE>
__device__ __forceinline__ int rd(const int *x) {
  if (IN_PLACE) return *x;
  return __ldg(x);
}

template <bool IN_PLACE>
__global__ void __launch_bounds__(PT) k_kv_plan(const pk_kv_plan_args p, int page_shift) {
  extern __shared__ uint32_t at[];
  __shared__ Pair sums[PW];
  pdl_trigger();
  pdl_wait();
  const int S = p.n_seq, tid = threadIdx.x;
  uint32_t *start = at, *take = at + S + 1, *back = at + 2 * (S + 1);
  auto held_of = [&](int s) { return min(max(rd<IN_PLACE>(p.held + s), 0), p.max_pages); };
  auto shared_of = [&](int s) { return p.shared ? min(max(__ldg(p.shared + s), 0), held_of(s)) : 0; };
  auto is_done = [&](int s) { return p.done && __ldg(p.done + s) != 0; };
  // (written in place behind the barrier)
  const int n_free = min(max(rd<IN_PLACE>(p.n_free), 0), p.free_cap);
  for (int s = tid; s < S; s += PT) {
    const int n = min(max(__ldg(p.n_new + s), 0), p.n_tok);
    start[s] = is_done(s) || __ldg(p.ctx + s) < 0 ? 0u : (uint32_t)n;
  }
  __syncthreads();
  // a run of slots a thread, of odd length so that the threads' places are in different banks
  const int run = ((S + PT - 1) / PT) | 1, s0 = min(S, tid * run), s1 = min(S, s0 + run);
  Pair v{0, 0}, total;
  for (int s = s0; s < s1; s++) v.a = add_to(v.a, start[s], (uint32_t)p.n_tok);
  v = scan2(v, (uint32_t)p.n_tok, sums, total);
  for (int s = s0; s < s1; s++) {
    const uint32_t n = start[s];
    start[s] = v.a;
    v.a = add_to(v.a, n, (uint32_t)p.n_tok);
  }
  if (tid == 0) start[S] = total.a;
  const int n_used = (int)total.a;
  __syncthreads();
  for (int s = tid; s < S; s += PT) {
    const int n = (int)(start[s + 1] - start[s]), held = held_of(s);
    const long long last = (long long)__ldg(p.ctx + s) + n + p.page_size - 1;
    const int need = n > 0 ? (int)min(last >> page_shift, (long long)p.max_pages) : 0;
    take[s] = (uint32_t)max(need - held, 0);
    back[s] = is_done(s) ? (uint32_t)(held - shared_of(s)) : 0u;
  }
  __syncthreads();
  v = {0, 0};
  const uint32_t none = 0xffffffffu;  // (n_seq * max_pages is below 2^31)
  for (int s = s0; s < s1; s++) v.a += take[s], v.b += back[s];
  v = scan2(v, none, sums, total);
  for (int s = s0; s < s1; s++) {
    const uint32_t a = take[s], b = back[s];
    take[s] = v.a;
    back[s] = v.b;
    v.a += a;
    v.b += b;
  }
  if (tid == 0) take[S] = total.a, back[S] = total.b;
  __syncthreads();
  const long long have = (long long)n_free + total.b, taken = total.a;  // entries of the list; pages asked for
  const long long left = max(have - taken, 0LL);
  const int kept = (int)min(left, (long long)p.free_cap);
  auto entry = [&](long long i) {  // of the list, 0 <= i < have
    if (i < n_free) return rd<IN_PLACE>(p.free + i);
    const uint32_t x = (uint32_t)(i - n_free);
    const int s = last_at(back, S, x);
    return rd<IN_PLACE>(p.pages + (size_t)s * p.max_pages + shared_of(s) + (x - back[s]));
  };
  auto page_taken = [&](uint32_t k) { return k < have ? entry(have - 1 - k) : -1; };

  const int cta = blockIdx.x, ctas = gridDim.x;
  const long long g0 = (long long)cta * PT + tid, step = (long long)ctas * PT;
  // the tokens
  if (p.pos || p.seq || p.slot) {
    for (long long t = g0; t < p.n_tok; t += step) {
      int pos = 0, seq = -1;
      long long slot = -1;
      if (t < n_used) {
        seq = last_at(start, S, (uint32_t)t);
        const long long at = __ldg(p.ctx + seq) + (t - start[seq]), j = at >> page_shift;
        pos = (int)min(at, 0x7fffffffLL);
        if (j < p.max_pages && at <= 0x7fffffffLL && p.slot) {
          const int held = held_of(seq);
          const int page = j < held ? rd<IN_PLACE>(p.pages + (size_t)seq * p.max_pages + j) : page_taken(take[seq] + (uint32_t)(j - held));
          if (page >= 0) slot = ((long long)page << page_shift) + (pos & (p.page_size - 1));
        }
      }
      if (p.pos) p.pos[t] = pos;
      if (p.seq) p.seq[t] = seq;
      if (p.slot) p.slot[t] = slot;
    }
  }
  // the pages taken
  for (long long k = g0; k < taken; k += step) {
    const int s = last_at(take, S, (uint32_t)k);
    p.pages_out[(size_t)s * p.max_pages + held_of(s) + (k - take[s])] = page_taken((uint32_t)k);
  }
  // the list; in place only what changes, entries that others may read being left for later
  for (long long i = (IN_PLACE ? n_free : 0) + g0; i < (IN_PLACE ? kept : p.free_cap); i += step)
    p.free_out[i] = i < kept ? entry(i) : i < n_free ? -1 : __ldg(p.free + i);
  // the tables' other entries
  if (!IN_PLACE) {
    // a warp takes 1024 entries of a row at a time
    const int lane = tid & 31, segs = (p.max_pages + 1023) / 1024;
    const bool vec = (p.max_pages & 3) == 0 && (((uintptr_t)p.pages | (uintptr_t)p.pages_out) & 15) == 0;
    for (long long x = (long long)cta * PW + (tid >> 5); x < (long long)S * segs; x += (long long)ctas * PW) {
      const int s = (int)(x / segs), j0 = (int)(x - (long long)s * segs) * 1024, j1 = min(j0 + 1024, p.max_pages);
      const int held = held_of(s), fresh = held + (int)(take[s + 1] - take[s]);
      const bool done = is_done(s);
      const int *from = p.pages + (size_t)s * p.max_pages;
      int *to = p.pages_out + (size_t)s * p.max_pages;
      if (vec) {
#pragma unroll 4
        for (int j = j0 + 4 * lane; j < j1; j += 128) {
          int4 w = __ldg(reinterpret_cast<const int4 *>(from + j));
          if (done) {
            w.x = j < held ? -1 : w.x, w.y = j + 1 < held ? -1 : w.y, w.z = j + 2 < held ? -1 : w.z, w.w = j + 3 < held ? -1 : w.w;
          }
          if (j + 4 <= held || j >= fresh) {
            *reinterpret_cast<int4 *>(to + j) = w;
          } else {
            if (j < held || j >= fresh) to[j] = w.x;
            if (j + 1 < held || j + 1 >= fresh) to[j + 1] = w.y;
            if (j + 2 < held || j + 2 >= fresh) to[j + 2] = w.z;
            if (j + 3 < held || j + 3 >= fresh) to[j + 3] = w.w;
          }
        }
      } else {
        for (int j = j0 + lane; j < j1; j += 32)
          if (j < held || j >= fresh) to[j] = done && j < held ? -1 : __ldg(from + j);
      }
    }
  }
  if (cta == 0)
    for (int s = tid; s <= S; s += PT) p.start[s] = (int)start[s];
  if (IN_PLACE) {
    // a cluster is all of the grid: from here on nobody reads an input that is written
    asm volatile("barrier.cluster.arrive.release.aligned;\n barrier.cluster.wait.acquire.aligned;" ::: "memory");
    for (long long i = kept + g0; i < n_free; i += step) p.free_out[i] = -1;
  }
  // (which slots' counts are whose: each thread reads its own slots' before it writes them)
  const int lane = tid & 31;
  for (long long s = (long long)cta * PW + (tid >> 5); s < S; s += (long long)ctas * PW) {
    const int held = held_of((int)s);
    const bool done = is_done((int)s);
    if (IN_PLACE && done)
      for (int j = lane; j < held; j += 32) p.pages_out[(size_t)s * p.max_pages + j] = -1;
    const long long k0 = take[s], k1 = take[s + 1];
    __syncwarp();
    if (lane == 0) p.held_out[s] = done ? 0 : held + (int)(min(k1, max(have, k0)) - k0);
  }
  if (g0 == 0) {
    *p.lacking = (int)min(max(taken - have, 0LL), 0x7fffffffLL);
    *p.n_free_out = kept;
  }
}

}  // namespace

cudaError_t launch_kv_plan(const pk_kv_plan_args &p, bool in_place, cudaStream_t st) {
  int shift = 0;
  while ((1 << shift) < p.page_size) shift++;
  const int smem = 3 * (p.n_seq + 1) * (int)sizeof(uint32_t);
  if (in_place)
    // (one CTA's sums are as long as eight's: few slots and tokens take one)
    return launch_cluster(k_kv_plan<true>, 8, dim3(8), dim3(PT), smem, st, p, shift);
  // a CTA for 4096 entries copied or 512 tokens, up to two an SM
  const long long work = ((long long)p.n_seq * p.max_pages + p.free_cap) / 4096 + p.n_tok / PT + 1;
  return launch(k_kv_plan<false>, dim3((unsigned)std::min(work, 296LL)), dim3(PT), smem, st, p, shift);
}

}  // namespace pk
