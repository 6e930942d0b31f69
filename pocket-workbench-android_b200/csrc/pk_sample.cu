// pk_sample.cu -- a token for every row of logits, from given random numbers
// (pk_sample_rows): temperature, min-p, top-k and top-p.  pk_sample takes one
// row in the reference's order of operations (sampler.rs:21-92), with its sort.
//
//   w_t = 2^(y_t), y_t = (x_t - max x) log2(e) / temp;  order: x down, index up
// All three rules keep a beginning of that order, so what is kept is everything
// down to one (logit, index), the cut.  Without a sort of the row:
//   1  the first token (largest logit, lowest index): y <= 0.  min_p is a least
//      logit.
//   2  a histogram of y in steps of a 16th of a nat: how many tokens, and their
//      weight, in f32 as the parts by which they exceed the bin's lowest weight
//      (sums within 2^-17 of right; a 4e-5th is allowed for).  Its sums from the
//      top say which bins hold the cut.
//   3  the tokens of those bins (or of all bins down to there, if they are few,
//      for top-k and top-p at once) are sorted and added up exactly, beginning
//      with the exact weight above them.  If they are too many, as in rows of
//      equal logits, halving steps on (logit, index) come before.
//   4  sums of the kept weights by index, the token in whose part u falls.
// A token depends on sums of a whole vocabulary next to whose borders u may lie:
// at 128256 borders an error of 2^-24 would change one token in a hundred.  So
// weights are made in double (a table of 16 and five terms of the series for
// 2^r: 1.4e-13) and added as 64-bit integers, in which no order matters; they
// are 2^-q steps of the largest, n 2^q <= 2^62.
//
// A row is read once, into the shared memory of a cluster of up to 8 CTAs
// (three CTAs an SM up to 64 KB each), and gone over there; rows that do not fit
// are read again each time.
#include <math_constants.h>

#include <algorithm>

#include "pk_cache.cuh"
#include "pk_cache.h"
#include "pk_launch.h"

namespace pk {
namespace {

typedef unsigned long long u64;

constexpr int ST = 512, SW = ST / 32;  // threads, warps
constexpr int BINS = 1024, CAP = 480;  // of the histogram; tokens that are sorted (three CTAs with 64144 bytes of a row fit an SM)
static_assert(2 * BINS * sizeof(uint32_t) >= ST * sizeof(u64), "room to sort");
static_assert(BINS == 2 * ST && CAP <= ST, "two bins and one sorted token a thread");
constexpr float MARGIN = 4e-5f;
constexpr int LAST = 0x7fffffff;

struct SampleK {
  const void *logits;
  long long stride;
  int n, cluster, seg;   // seg: positions a CTA, whole 16-byte vectors
  int q;                 // fixed-point bits of a weight
  float part, margin;    // steps of a bin's excess; what the histogram's sums may be off by
  pk_sample_args p;
};

struct Smem {  // behind the row's values
  uint32_t cnt[BINS], part[BINS];
  u64 cand[CAP];
  double table[16];
  u64 warp[SW], x[6];   // of the CTA's warps; what the cluster's CTAs tell each other
  uint32_t warp2[SW], n_cand, lo, hi, at;
  float warpf[SW], cut_x, least;
  int cut_i;
};

__device__ __forceinline__ uint32_t key_of(float x) {  // ascending
  const uint32_t u = __float_as_uint(x + 0.0f);  // (-0 is 0)
  return u ^ ((uint32_t)((int)u >> 31) | 0x80000000u);
}
__device__ __forceinline__ float of_key(uint32_t k) { return __uint_as_float(k & 0x80000000u ? k ^ 0x80000000u : ~k); }
__device__ __forceinline__ u64 order_of(float x, int i) { return (u64)key_of(x) << 32 | (uint32_t)~i; }

__device__ __forceinline__ uint32_t map_rank(uint32_t a, int rank) {
  uint32_t r;
  asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(rank));
  return r;
}
__device__ __forceinline__ u64 peer64(const void *p, int rank) {
  u64 v;
  asm volatile("ld.shared::cluster.u64 %0, [%1];" : "=l"(v) : "r"(map_rank(shaddr(p), rank)) : "memory");
  return v;
}
__device__ __forceinline__ uint32_t peer32(const void *p, int rank) {
  uint32_t v;
  asm volatile("ld.shared::cluster.u32 %0, [%1];" : "=r"(v) : "r"(map_rank(shaddr(p), rank)) : "memory");
  return v;
}

// 16 bytes of a row as f32, NaN as -inf.
template <class E> constexpr int VE = 16 / (int)sizeof(E);
template <class E>
__device__ __forceinline__ void values(uint4 w, float (&x)[VE<E>]) {
  const E *e = reinterpret_cast<const E *>(&w);
#pragma unroll
  for (int i = 0; i < VE<E>; i++) x[i] = fmaxf(to_f(e[i]), -CUDART_INF_F);
}
template <class E> __device__ __forceinline__ E minus_inf() { return from_f<E>(-CUDART_INF_F); }

template <class E, bool BIG>
struct Row {
  static constexpr int V = VE<E>;
  const SampleK &a;
  Smem &sm;
  const E *base;    // the row
  const uint4 *data;  // the CTA's positions in shared memory
  int tid, lane, warp, rank, shift, end;  // position p is token p - shift; positions of this row: shift .. end - 1
  int p0, vecs, per;  // this CTA's first position, its vectors, those of a warp (its own run of them)
  float top;        // the largest logit
  double scale;     // log2(e) / temp
  float cx;         // the cut: kept is what is larger, or equal with an index up to ci
  int ci;

  __device__ __forceinline__ void sync() const {
    if (a.cluster == 1) __syncthreads();
    else asm volatile("barrier.cluster.arrive.release.aligned;\n barrier.cluster.wait.acquire.aligned;" ::: "memory");
  }
  __device__ __forceinline__ E load(long long p) const { return p >= shift && p < end ? base[p - shift] : minus_inf<E>(); }
  __device__ __forceinline__ void vec(int i, float (&x)[V]) const {  // vector i of this CTA
    if (BIG) {
#pragma unroll
      for (int e = 0; e < V; e++) x[e] = fmaxf(to_f(load((long long)p0 + (long long)i * V + e)), -CUDART_INF_F);
    } else {
      values<E>(data[i], x);
    }
  }
  // f(value, token) for this thread's values, in order
  template <class F>
  __device__ __forceinline__ void each(F f) const {
    const int w1 = min(vecs, (warp + 1) * per);
    for (int i = warp * per + lane; i < w1; i += 32) {
      float x[V];
      vec(i, x);
#pragma unroll
      for (int e = 0; e < V; e++) f(x[e], p0 + i * V + e - shift);
    }
  }
  // the same for whole warps: f is called by all lanes, with -inf past the end
  template <class F>
  __device__ __forceinline__ void each_warp(F f) const {
    const int w1 = min(vecs, (warp + 1) * per);
    for (int i0 = warp * per; i0 < w1; i0 += 32) {
      float x[V];
      const int i = i0 + lane;
      if (i < w1) {
        vec(i, x);
      } else {
#pragma unroll
        for (int e = 0; e < V; e++) x[e] = -CUDART_INF_F;
      }
      f(x, p0 + i * V - shift);
    }
  }
  __device__ __forceinline__ bool kept(float x, int i) const { return x > cx || (x == cx && i <= ci); }

  // 2^y of the weight, times 2^up (y <= 0)
  __device__ __forceinline__ double weight(float x, int up) const {
    double y = ((double)x - (double)top) * scale;
    if (x == top) y = 0.0;
    if (!(y > -64.0)) return 0.0;
    const double magic = 6755399441055744.0;  // 1.5 * 2^52: the sum's low bits are the rounded integer
    const double t = fma(y, 16.0, magic);
    const int k = __double2loint(t);
    const double r = fma(t - magic, -0.0625, y);
    double f = 0.0013333558146428443;  // ln(2)^i / i!
    f = fma(f, r, 0.009618129107628477);
    f = fma(f, r, 0.05550410866482158);
    f = fma(f, r, 0.24022650695910072);
    f = fma(f, r, 0.6931471805599453);
    f = fma(f, r, 1.0) * sm.table[k & 15];
    return __hiloint2double(__double2hiint(f) + (((k >> 4) + up) << 20), __double2loint(f));
  }
  __device__ __forceinline__ u64 fixed(float x) const {
    const double w = weight(x, a.q) + 4503599627370496.0;  // 2^52
    return (u64)__double_as_longlong(w) - 0x4330000000000000ull;
  }
  // bin of y, and the place in it (0 .. 1)
  __device__ __forceinline__ int bin(float x, float per_unit, float &place) const {
    const float d = x == top ? 0.0f : (top - x) * per_unit;
    const float b = floorf(fminf(d, (float)(BINS - 1)));  // (NaN: the last)
    place = fminf(d - b, 1.0f);
    return (int)b;
  }

  __device__ __forceinline__ u64 sum_warp(u64 v) const {
#pragma unroll
    for (int i = 16; i > 0; i >>= 1) v += __shfl_xor_sync(0xffffffffu, v, i);
    return v;
  }
  // sum of the CTA's threads into slot x[i] (for the cluster, behind sync())
  __device__ __forceinline__ void sum_to(u64 v, int i) const {
    v = sum_warp(v);
    if (lane == 0) sm.warp[warp] = v;
    __syncthreads();
    if (warp == 0) {
      v = sum_warp(lane < SW ? sm.warp[lane] : 0);
      if (lane == 0) sm.x[i] = v;
    }
  }
  __device__ __forceinline__ u64 all_sum(int i) const { return sum_warp(lane < a.cluster ? peer64(&sm.x[i], lane) : 0); }
  // exclusive sums over the CTA's threads
  __device__ __forceinline__ u64 scan(u64 v) const {
    u64 x = v;
#pragma unroll
    for (int i = 1; i < 32; i *= 2) {
      const u64 y = __shfl_up_sync(0xffffffffu, x, i);
      if (lane >= i) x += y;
    }
    if (lane == 31) sm.warp[warp] = x;
    __syncthreads();
    u64 before = 0;
    for (int w = 0; w < warp; w++) before += sm.warp[w];
    __syncthreads();
    return before + x - v;
  }
};

template <class E, bool BIG>
__global__ void __launch_bounds__(ST, BIG ? 2 : 3) k_sample(const SampleK a) {
  constexpr int V = VE<E>;
  extern __shared__ __align__(16) uint8_t smem[];
  Smem &sm = *reinterpret_cast<Smem *>(smem + (BIG ? 0 : (size_t)a.seg * sizeof(E)));
  const int row = blockIdx.x / a.cluster, rank = blockIdx.x % a.cluster;
  const E *base = reinterpret_cast<const E *>(a.logits) + row * a.stride;
  const int shift = (int)(((uintptr_t)base / sizeof(E)) % V);
  const long long first = (long long)rank * a.seg, all = (long long)a.n + shift;
  const int mine = (int)max(0LL, min((long long)a.seg, all - first));
  const int vecs = (mine + V - 1) / V, per = (vecs + SW - 1) / SW;
  Row<E, BIG> r{a, sm, base, reinterpret_cast<const uint4 *>(smem), (int)threadIdx.x, (int)threadIdx.x & 31, (int)threadIdx.x >> 5, rank, shift, (int)all,
                (int)first, vecs, (per + 31) / 32 * 32, 0.0f, 0.0, 0.0f, LAST};
  const int tid = r.tid, lane = r.lane, warp = r.warp;
  pdl_trigger();
  pdl_wait();
  if (!BIG) {
    const uint32_t to = shaddr(smem);
    for (int i = tid; i < vecs; i += ST) {
      const long long p = first + (long long)i * V;
      if (p >= shift && p + V <= all) {
        asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(to + 16 * i), "l"(base + (p - shift)) : "memory");
      } else {
        E *e = reinterpret_cast<E *>(smem) + i * V;
#pragma unroll
        for (int j = 0; j < V; j++) e[j] = r.load(p + j);
      }
    }
    asm volatile("cp.async.commit_group;" ::: "memory");
  }
  const float u = __ldg(a.p.u + row), temp = a.p.temp ? __ldg(a.p.temp + row) : 1.0f;
  const float top_p = a.p.top_p ? __ldg(a.p.top_p + row) : 1.0f, min_p = a.p.min_p ? __ldg(a.p.min_p + row) : 0.0f;
  const int top_k = a.p.top_k ? __ldg(a.p.top_k + row) : 0;
  if (tid < 16) sm.table[tid] = exp2((double)tid / 16.0);
  if (tid == 0) sm.n_cand = 0;
  sm.cnt[tid] = sm.cnt[tid + ST] = sm.part[tid] = sm.part[tid + ST] = 0;
  asm volatile("cp.async.wait_group 0;" ::: "memory");
  __syncthreads();

  // ---- 1: the first token
  int where = -1;
  {
    float best = -CUDART_INF_F;
    int at = LAST;
    r.each([&](float x, int i) {
      if (x > best) best = x, at = i;
    });
    const uint32_t k = __reduce_max_sync(0xffffffffu, key_of(best));
    const int i = (int)__reduce_min_sync(0xffffffffu, key_of(best) == k ? (uint32_t)at : (uint32_t)LAST);
    if (lane == 0) sm.warp[warp] = (u64)k << 32 | (uint32_t)~i;
    __syncthreads();
    auto most = [&](u64 v) {
#pragma unroll
      for (int j = 16; j > 0; j >>= 1) v = max(v, __shfl_xor_sync(0xffffffffu, v, j));
      return v;
    };
    if (warp == 0) {
      const u64 v = most(lane < SW ? sm.warp[lane] : 0);
      if (lane == 0) sm.x[0] = v;
    }
    r.sync();
    const u64 v = most(lane < a.cluster ? peer64(&sm.x[0], lane) : 0);
    r.top = of_key((uint32_t)(v >> 32));
    where = (int)~(uint32_t)v;
  }
  const bool empty = r.top == -CUDART_INF_F;
  if (empty || !(temp > 0.0f) || top_k == 1 || top_p <= 0.0f || min_p > 1.0f) {  // (the same for the whole cluster)
    if (rank == 0 && tid == 0) {
      a.p.tok[row] = empty ? -1 : where;
      if (a.p.prob) a.p.prob[row] = empty ? 0.0f : 1.0f;
      if (a.p.kept) a.p.kept[row] = empty ? 0 : 1;
    }
    r.sync();  // (others may be reading what this CTA told)
    return;
  }
  r.scale = 1.4426950408889634074 / (double)temp;
  r.cx = -CUDART_MAX_NORMAL_F;
  if (min_p > 0.0f) {
    if (tid == 0) {  // the least logit with y >= log2(min_p): a guess, then its neighbours
      const double least = log2((double)min_p);
      auto ok = [&](float x) { return x == r.top || ((double)x - (double)r.top) * r.scale >= least; };
      float g = r.top;
      if (r.top < CUDART_INF_F && r.scale > 0.0) g = fmaxf(fminf((float)((double)r.top + least / r.scale), r.top), -CUDART_MAX_NORMAL_F);
      if (r.top < CUDART_INF_F && r.scale == 0.0) g = -CUDART_MAX_NORMAL_F;
      for (int i = 0; i < 8 && !ok(g); i++) g = nextafterf(g, CUDART_INF_F);
      for (int i = 0; i < 8 && g > -CUDART_MAX_NORMAL_F && ok(nextafterf(g, -CUDART_INF_F)); i++) g = nextafterf(g, -CUDART_INF_F);
      sm.least = g;
    }
    __syncthreads();
    r.cx = sm.least;
  }

  // ---- 2, 3: the cut of top-k, then of top-p
  bool do_k = top_k > 0 && top_k < a.n, do_p = top_p < 1.0f;
  const float per_unit = fminf(16.0f / temp, 1e30f);
  for (bool again = false; do_k || do_p; again = true) {
    const bool weigh = !do_k;  // top-p of all that is kept: their exact weight
    if (again) {
      r.sync();  // (the histogram has been read)
      sm.cnt[tid] = sm.cnt[tid + ST] = sm.part[tid] = sm.part[tid + ST] = 0;
      if (tid == 0) sm.n_cand = 0;
      __syncthreads();
    }
    u64 sum = 0;
    r.each([&](float x, int i) {
      if (!r.kept(x, i)) return;
      float place;
      const int b = r.bin(x, per_unit, place);
      atomicAdd(&sm.cnt[b], 1u);
      if (do_p && b < BINS - 1) {
        // 2^((1 - place) / 16 nat) - 1, of the bin's lowest weight
        float over;
        asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(over) : "f"((1.0f - place) * (1.4426950408889634f / 16.0f)));
        atomicAdd(&sm.part[b], (uint32_t)__float2int_rn((over - 1.0f) * a.part));
      }
      if (weigh) sum += r.fixed(x);
    });
    if (weigh) r.sum_to(sum, 1);
    r.sync();
    const u64 weight = weigh ? r.all_sum(1) : 0;
    // bins 2 tid, 2 tid + 1 of the whole row, and the sums down to them
    uint32_t c[2] = {0, 0};
    float m[2] = {0.0f, 0.0f};
    for (int k = 0; k < a.cluster; k++) {
#pragma unroll
      for (int j = 0; j < 2; j++) {
        c[j] += peer32(&sm.cnt[2 * tid + j], k);
        if (do_p) m[j] += (float)peer32(&sm.part[2 * tid + j], k);
      }
    }
#pragma unroll
    for (int j = 0; j < 2; j++) {
      const int b = 2 * tid + j;
      m[j] = do_p && b < BINS - 1 ? exp2f((float)(b + 1) * (-1.4426950408889634f / 16.0f)) * fmaf(m[j], 1.0f / a.part, (float)c[j]) : 0.0f;
    }
    uint32_t cs = c[0] + c[1];
    float ms = m[0] + m[1];
#pragma unroll
    for (int i = 1; i < 32; i *= 2) {
      const uint32_t y = __shfl_up_sync(0xffffffffu, cs, i);
      const float z = __shfl_up_sync(0xffffffffu, ms, i);
      if (lane >= i) cs += y, ms += z;
    }
    if (lane == 31) sm.warp2[warp] = cs, sm.warpf[warp] = ms;
    if (tid == 0) sm.lo = sm.hi = BINS - 1;
    __syncthreads();
    uint32_t total = 0;
    float mass = 0.0f, mb = 0.0f;
    {
      uint32_t cb = 0;
      for (int w = 0; w < SW; w++) {
        if (w == warp) cb = total, mb = mass;
        total += sm.warp2[w];
        mass += sm.warpf[w];
      }
      cs += cb, ms += mb;
    }
    // of the first bin, and the second
    const uint32_t ce[2] = {cs - c[1], cs};
    const float me[2] = {ms - m[1], ms};
    const uint32_t k = min((uint32_t)top_k, total);
    if (do_k) {
#pragma unroll
      for (int j = 0; j < 2; j++)
        if (ce[j] >= k && ce[j] - c[j] < k) sm.lo = sm.hi = 2 * tid + j;
    } else {
      const float low = mass * top_p * (1.0f - a.margin), high = mass * top_p * (1.0f + a.margin);
      // (sums need not ascend by the last bit: the first bin that passes)
#pragma unroll
      for (int j = 0; j < 2; j++) {
        if (me[j] >= low) atomicMin(&sm.lo, (uint32_t)(2 * tid + j));
        if (me[j] >= high) atomicMin(&sm.hi, (uint32_t)(2 * tid + j));
      }
    }
    __syncthreads();
    const int hi = (int)sm.hi;
    int lo = (int)sm.lo;
#pragma unroll
    for (int j = 0; j < 2; j++) {
      if (2 * tid + j == hi) sm.at = ce[j];
      if (2 * tid + j == lo) sm.warp2[0] = ce[j] - c[j];
    }
    __syncthreads();
    const uint32_t down = sm.at;  // tokens down to bin hi
    uint32_t above = sm.warp2[0];  // before bin lo
    if (do_k && (uint32_t)top_k >= total && down > CAP) {  // top-k keeps them all
      do_k = false;
      continue;
    }
    const bool whole = down <= CAP;
    if (whole) lo = 0, above = 0;
    const bool both = do_k && do_p && whole;
    uint32_t inside = down - above;
    // (by bins, or after halving by order) is it in question? is it before?
    u64 o_lo = 0, o_hi = ~0ull, base_w = 0;
    bool by_order = false;
    auto side = [&](float x, int i) {  // 0: in question, 1: before, -1: behind
      if (by_order) {
        const u64 o = order_of(x, i);
        return o > o_hi ? 1 : o < o_lo ? -1 : 0;
      }
      float place;
      const int b = r.bin(x, per_unit, place);
      return b < lo ? 1 : b > hi ? -1 : 0;
    };
    const double target = (double)top_p * (double)weight;
    if (inside > CAP) {
      // Halving.  The order's bounds first, and the exact weight before them.
      u64 least = ~0ull, most = 0, before = 0;
      r.each([&](float x, int i) {
        if (!r.kept(x, i)) return;
        const int s = side(x, i);
        if (s == 0) least = min(least, order_of(x, i)), most = max(most, order_of(x, i));
        if (s > 0 && weigh) before += r.fixed(x);
      });
#pragma unroll
      for (int j = 16; j > 0; j >>= 1) least = min(least, __shfl_xor_sync(0xffffffffu, least, j)), most = max(most, __shfl_xor_sync(0xffffffffu, most, j));
      r.sum_to(before, 2);
      __syncthreads();
      if (tid == 0) sm.x[3] = ~0ull, sm.x[4] = 0;
      __syncthreads();
      if (lane == 0) atomicMin(&sm.x[3], least), atomicMax(&sm.x[4], most);
      r.sync();
      base_w = r.all_sum(2);
      for (int j = 0; j < a.cluster; j++) {
        const u64 x = peer64(&sm.x[3], j), y = peer64(&sm.x[4], j);
        if (j == 0 || x < o_lo) o_lo = x;
        if (j == 0 || y > o_hi) o_hi = y;
      }
      by_order = true;
      r.sync();  // (the slots are written again)
      for (int turn = 0; inside > CAP && turn < 64; turn++) {  // (orders differ: 63 at most)
        const u64 mid = o_lo + (o_hi - o_lo) / 2;
        u64 n_up = 0, w_up = 0;
        r.each([&](float x, int i) {
          if (!r.kept(x, i)) return;
          const u64 o = order_of(x, i);
          if (o > mid && o <= o_hi) {
            n_up++;
            if (weigh) w_up += r.fixed(x);
          }
        });
        // (slots in turn: a CTA may be a step ahead of one that still reads)
        const int at = 2 + (turn & 1);
        r.sum_to(n_up, at);
        __syncthreads();
        r.sum_to(w_up, at + 2);
        r.sync();
        n_up = r.all_sum(at);
        w_up = r.all_sum(at + 2);
        const bool up = do_k ? above + n_up >= k : (double)(base_w + w_up) >= target;
        if (up) {
          o_lo = mid + 1;
          inside = (uint32_t)n_up;
        } else {
          o_hi = mid;
          inside -= (uint32_t)n_up;
          above += (uint32_t)n_up;
          base_w += w_up;
        }
      }
      r.sync();
    }
    // the tokens in question to the first CTA, and the exact weight before them
    u64 before = 0;
    r.each_warp([&](const float (&x)[V], int i0) {
#pragma unroll
      for (int e = 0; e < V; e++) {
        const bool on = r.kept(x[e], i0 + e);
        const int s = on ? side(x[e], i0 + e) : -1;
        if (s > 0 && weigh && !by_order) before += r.fixed(x[e]);
        const uint32_t lanes = __ballot_sync(0xffffffffu, s == 0);
        if (lanes) {
          uint32_t at = 0;
          if (lane == __ffs(lanes) - 1)
            asm volatile("atom.relaxed.cluster.shared::cluster.add.u32 %0, [%1], %2;" : "=r"(at) : "r"(map_rank(shaddr(&sm.n_cand), 0)), "r"(__popc(lanes)) : "memory");
          at = __shfl_sync(0xffffffffu, at, __ffs(lanes) - 1) + __popc(lanes & ((1u << lane) - 1));
          if (s == 0 && at < CAP)
            asm volatile("st.shared::cluster.u64 [%0], %1;" ::"r"(map_rank(shaddr(&sm.cand[0]), 0) + at * 8), "l"(order_of(x[e], i0 + e)) : "memory");
        }
      }
    });
    if (weigh && !by_order) r.sum_to(before, 5);
    r.sync();
    if (rank == 0) {
      if (weigh && !by_order) base_w = r.all_sum(5);
      const int nc = min((int)sm.n_cand, CAP);
      u64 v = tid < nc ? sm.cand[tid] : 0;
      u64 *swap = reinterpret_cast<u64 *>(sm.cnt);  // (the histogram has been read)
      int n2 = 32;
      while (n2 < nc) n2 *= 2;
      for (int size = 2; size <= n2; size *= 2)
        for (int j = size / 2; j > 0; j /= 2) {
          u64 o;
          if (j >= 32) {
            swap[tid] = v;
            __syncthreads();
            o = swap[tid ^ j];
            __syncthreads();
          } else {
            o = __shfl_xor_sync(0xffffffffu, v, j);
          }
          const bool down_here = (tid & size) == 0, low_half = (tid & j) == 0;
          v = down_here == low_half ? max(v, o) : min(v, o);
        }
      const float x = of_key((uint32_t)(v >> 32));
      // the last one that top-k leaves
      const int most = do_k ? min(nc, (int)(k - above)) : nc;
      int cut = most - 1;
      if (!do_k || both) {
        const u64 w = tid < most ? r.fixed(x) : 0, b = r.scan(w);
        double goal = target;
        if (both) {
          if (tid == ST - 1) sm.x[5] = b + w;
          __syncthreads();
          goal = (double)top_p * (double)sm.x[5];
        }
        if (tid == 0) sm.at = (uint32_t)cut;
        __syncthreads();
        if (tid < most && (double)(base_w + b + w) >= goal && (tid == 0 || (double)(base_w + b) < goal)) sm.at = (uint32_t)tid;
        __syncthreads();
        cut = (int)sm.at;
      }
      if (tid == cut) sm.cut_x = x, sm.cut_i = (int)~(uint32_t)v;
    }
    r.sync();
    r.cx = __uint_as_float(peer32(&sm.cut_x, 0));
    r.ci = (int)peer32(&sm.cut_i, 0);
    if (do_k && !both) do_k = false;
    else do_k = do_p = false;
  }

  // ---- 4: the kept weights by index
  u64 sum = 0;
  uint32_t n = 0;
  r.each([&](float x, int i) {
    if (!r.kept(x, i)) return;
    n++;
    sum += r.fixed(x);
  });
  const u64 mine_w = r.sum_warp(sum);
  n = __reduce_add_sync(0xffffffffu, n);
  __syncthreads();  // (sums of before have been read)
  if (lane == 0) sm.warp[warp] = mine_w, sm.warp2[warp] = n;
  __syncthreads();
  if (warp == 0) {
    const u64 w = r.sum_warp(lane < SW ? sm.warp[lane] : 0);
    const uint32_t c = __reduce_add_sync(0xffffffffu, lane < SW ? sm.warp2[lane] : 0);
    if (lane == 0) sm.x[2] = w, sm.x[3] = c;  // (another CTA may still read x[0])
  }
  r.sync();
  u64 all_w = 0, before = 0, all_n = 0;
  for (int j = 0; j < a.cluster; j++) {
    if (j == rank) before = all_w;
    all_w += peer64(&sm.x[2], j);
    all_n += peer64(&sm.x[3], j);
  }
  // the first token whose sum passes floor(u W) passes u W (u below 0 and NaN: the first)
  const double goal = (double)u * (double)all_w;
  u64 pass = goal > 0.0 ? (goal < 9.2e18 ? (u64)goal : all_w) : 0;
  pass = min(pass, all_w - 1);
  u64 from = before;
  for (int w = 0; w < warp; w++) from += sm.warp[w];
  if (pass >= from && pass < from + mine_w) {  // one warp of one CTA
    r.each_warp([&](const float (&x)[V], int i0) {
      u64 w[V], lanes = 0;
#pragma unroll
      for (int e = 0; e < V; e++) {
        w[e] = r.kept(x[e], i0 + e) ? r.fixed(x[e]) : 0;
        lanes += w[e];
      }
      u64 upto = lanes;
#pragma unroll
      for (int i = 1; i < 32; i *= 2) {
        const u64 y = __shfl_up_sync(0xffffffffu, upto, i);
        if (lane >= i) upto += y;
      }
      u64 b = from + upto - lanes;
#pragma unroll
      for (int e = 0; e < V; e++) {
        if (pass >= b && pass < b + w[e]) {
          a.p.tok[row] = i0 + e;
          if (a.p.prob) a.p.prob[row] = (float)(r.weight(x[e], a.q) / (double)all_w);
          if (a.p.kept) a.p.kept[row] = (int)all_n;
        }
        b += w[e];
      }
      from += __shfl_sync(0xffffffffu, upto, 31);
    });
  }
  r.sync();  // (others may be reading what this CTA told)
}

}  // namespace

cudaError_t launch_sample(const void *logits, int type, int rows, int n, long stride, const pk_sample_args &p, cudaStream_t st) {
  const int es = type == T_F32 ? 4 : 2, v = 16 / es;
  SampleK a{};
  a.logits = logits;
  a.stride = stride;
  a.n = n;
  a.p = p;
  int bits = 0;
  while ((1LL << bits) < n) bits++;
  a.q = std::min(50, 62 - bits);
  // CTAs a row: three fit an SM with 64 KB each, one with 208; more where the rows leave SMs without any
  const long long vecs = ((long long)n + 2 * v - 2) / v, most = 64 * 1024 / 16, wide = 208 * 1024 / 16;
  long long c = std::min(8LL, (vecs + most - 1) / most);
  while (c < 8 && rows * c * 2 <= 148 && vecs >= 512 * c) c *= 2;
  c = std::min(c, 8LL);
  const long long seg = (vecs + c - 1) / c;
  const bool big = seg > wide;
  a.cluster = (int)c;
  a.seg = (int)(seg * v);
  a.part = 2097152.0f;  // 2^21: an excess is below 2^-3.95, so 16384 of a bin and CTA fit 32 bits
  for (long long x = 16384; x < a.seg; x *= 2) a.part *= 0.5f;
  a.margin = MARGIN + 2.0f / a.part;
  const int smem = (int)sizeof(Smem) + (big ? 0 : (int)(seg * 16));
  const dim3 grid((unsigned)(rows * c)), block(ST);
#define GO(E) launch_cluster(big ? k_sample<E, true> : k_sample<E, false>, (int)c, grid, block, smem, st, a)
  return type == T_F32 ? GO(float) : type == T_F16 ? GO(__half) : GO(__nv_bfloat16);
#undef GO
}

}  // namespace pk
