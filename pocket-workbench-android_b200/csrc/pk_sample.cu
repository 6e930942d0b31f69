// pk_sample.cu -- a token for every row of logits, from given random numbers
// (pk_sample_rows): temperature, min-p, top-k and top-p.  pk_sample takes one
// row in the reference's order of operations (sampler.rs:21-92), with its sort.
//
//   w_t = 2^(y_t), y_t = (x_t - max x) log2(e) / temp;  order: x down, index up
// All three rules keep a beginning of that order, so what is kept is everything
// down to one (logit, index), the cut.  Without a sort of the row:
//   1  the largest logit: y <= 0.  min_p is a least logit.
//   2  a histogram of y in steps of a 16th of a nat: of tokens for top-k, for
//      top-p of their weights as multiples of the bin's lowest, in 2^-15 (a 6e-5th
//      is allowed for that and f32's logarithms).  Its sums from the top say
//      which bins hold the cut.
//   3  the tokens of those bins (or of all bins down to there, if they are few,
//      for top-k and top-p at once) are sorted and added up exactly, beginning
//      with the exact weight above them.  If they are too many, as in rows of
//      equal logits, halving steps on (logit, index) come before.
//   4  sums of the kept weights by index, the token in whose part u falls.
// A token depends on sums of a whole vocabulary next to whose borders u may lie:
// at 128256 borders an error of 2^-24 would change one token in a hundred.  So
// weights are made in double, 2^y from a table of 256 and three terms of the
// series (1.4e-13), and added as 64-bit integers, in which no order matters:
// 2^-q steps of the largest, n 2^q <= 2^62.
//
// A row is read once, into the shared memory of a cluster of up to 8 CTAs, and
// gone over there; rows that do not fit are read again each time.
#include <math_constants.h>

#include <algorithm>

#include "pk_cache.cuh"
#include "pk_cache.h"
#include "pk_launch.h"

namespace pk {
namespace {

typedef unsigned long long u64;

constexpr int ST = 512, SW = ST / 32;  // threads, warps
constexpr int BINS = 512, CAP = 512;   // of the histogram; tokens that are sorted
static_assert(BINS == ST && CAP == ST, "a bin and a sorted token a thread");
constexpr float MARGIN = 6e-5f;
constexpr int LAST = 0x7fffffff;
constexpr float MAXF = 3.402823466e38f;

struct SampleK {
  const void *logits;
  long long stride;
  int n, cluster, seg;   // seg: positions a CTA, whole 16-byte vectors
  int q;                 // fixed-point bits of a weight
  float unit, margin;    // a bin's lowest weight in the histogram; what its sums may be off by
  pk_sample_args p;
};

struct Smem {  // behind the row's values
  uint32_t hist[2][BINS];  // of even and of odd lanes, which then collide less
  u64 cand[CAP];
  double table[256];
  u64 warp[SW], x[6];   // of the CTA's warps; what the cluster's CTAs tell each other
  double off_min, off_low;
  uint32_t warp2[SW], n_cand, lo, hi, at, above, first;
  float warpf[SW], cut_x;
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

template <class E> constexpr int VE = 16 / (int)sizeof(E);

template <class E, bool BIG>
struct Row {
  static constexpr int V = VE<E>;
  const SampleK &a;
  Smem &sm;
  const E *base;      // the row
  const uint4 *data;  // the CTA's positions in shared memory
  int tid, lane, warp;
  int shift, end;     // position p is token p - shift; positions of this row: shift .. end - 1
  int p0, vecs, per;  // this CTA's first position, its vectors, those of a warp (its own run of them)
  float top = 0.0f, low = 0.0f;  // the largest logit; what is below `low` has no weight
  double step = 0.0, zero = 0.0;  // 256 log2(e) / temp; 1.5 * 2^52 less the largest logit's steps
  double scale = 0.0;  // log2(e) / temp
  bool exact = false;  // steps of logits themselves would lose bits: those of their differences
  float cx = 0.0f;     // the cut: kept is what is larger, or equal with an index up to ci
  int ci = LAST;

  __device__ __forceinline__ void sync() const {
    if (a.cluster == 1) __syncthreads();
    else asm volatile("barrier.cluster.arrive.release.aligned;\n barrier.cluster.wait.acquire.aligned;" ::: "memory");
  }
  __device__ __forceinline__ E load(long long p) const { return p >= shift && p < end ? base[p - shift] : from_f<E>(-CUDART_INF_F); }
  __device__ __forceinline__ void vec(int i, float (&x)[V]) const {  // vector i of this CTA
    if (BIG) {
#pragma unroll
      for (int e = 0; e < V; e++) x[e] = to_f(load((long long)p0 + (long long)i * V + e));
    } else {
      const uint4 w = data[i];
      const E *v = reinterpret_cast<const E *>(&w);
#pragma unroll
      for (int e = 0; e < V; e++) x[e] = to_f(v[e]);
    }
  }
  // f(four values, the first's token) for this thread's, in order.  NaN compares as false everywhere.
  template <class F>
  __device__ __forceinline__ void each4(F f) const {
    const int w1 = min(vecs, (warp + 1) * per);
    for (int i = warp * per + lane; i < w1; i += 32) {
      float x[V];
      vec(i, x);
#pragma unroll
      for (int e = 0; e < V; e += 4) f(x + e, p0 + i * V + e - shift);
    }
  }
  template <class F>
  __device__ __forceinline__ void each(F f) const {
    each4([&](const float *x, int i) {
#pragma unroll
      for (int e = 0; e < 4; e++) f(x[e], i + e);
    });
  }
  __device__ __forceinline__ bool kept(float x, int i) const { return x >= cx && (x > cx || i <= ci); }

  // The weight times 2^q (and a factor within 2^(1/512) of 1, the same for the
  // whole row), for low <= x <= top.  Where +inf is the largest, everything
  // below has none (low).
  __device__ __forceinline__ double weight(float x) const {
    double v;
    if (exact) {
      v = x == top ? 0.0 : ((double)x - (double)top) * scale;
    } else {  // x in double without the conversion, of which an SM makes 16 a cycle; 0 and subnormals become up to 2^-126
      const int u = __float_as_int(x);
      v = __hiloint2double(((u >> 3) & 0x8fffffff) + (896 << 20), u << 29);
    }
    const double t = fma(v, step, zero);  // its low bits are the number of steps, rounded
    const double r = fma(v, step, zero - t);  // what is left of them, -0.5 .. 0.5
    const int k = __double2loint(t);
    double f = 3.308302680541371e-09;  // (ln(2) / 256)^i / i!
    f = fma(f, r, 3.665565596910106e-06);
    f = fma(f, r, 0.0027076061740622863);
    f = fma(f, r, 1.0) * sm.table[k & 255];
    return __hiloint2double(__double2hiint(f) + ((k & ~255) << 12), __double2loint(f));
  }
  // the same, rounded to an integer
  static constexpr u64 ONE = 0x4330000000000000ull;  // 2^52's bits
  __device__ __forceinline__ u64 made(float x) const { return (u64)__double_as_longlong(weight(x) + 4503599627370496.0) - ONE; }
  __device__ __forceinline__ u64 fixed(float x) const { return x >= low ? made(x) : 0; }
  // of four those that are `on`
  __device__ __forceinline__ void add4(const float *x, const bool (&on)[4], u64 &sum) const {
    if (!(on[0] || on[1] || on[2] || on[3])) return;
#pragma unroll
    for (int e = 0; e < 4; e++) {
      const u64 w = made(on[e] ? x[e] : top);
      if (on[e]) sum += w;
    }
  }
  __device__ __forceinline__ u64 sum_kept(const float *x, int i) const {
    const float least = fmaxf(cx, low);
    bool on[4];
#pragma unroll
    for (int e = 0; e < 4; e++) on[e] = x[e] >= least && (x[e] > cx || i + e <= ci);
    u64 sum = 0;
    add4(x, on, sum);
    return sum;
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
__global__ void __launch_bounds__(ST, 2) k_sample(const SampleK a) {
  constexpr int V = VE<E>;
  extern __shared__ __align__(16) uint8_t smem[];
  Smem &sm = *reinterpret_cast<Smem *>(smem + (BIG ? 0 : (size_t)a.seg * sizeof(E)));
  const int row = blockIdx.x / a.cluster, rank = blockIdx.x % a.cluster;
  const E *base = reinterpret_cast<const E *>(a.logits) + row * a.stride;
  const int shift = (int)(((uintptr_t)base / sizeof(E)) % V);
  const long long first = (long long)rank * a.seg, all = (long long)a.n + shift;
  const int mine = (int)max(0LL, min((long long)a.seg, all - first));
  const int vecs = (mine + V - 1) / V, per = (vecs + SW - 1) / SW;
  Row<E, BIG> r{a, sm, base, reinterpret_cast<const uint4 *>(smem), (int)threadIdx.x, (int)threadIdx.x & 31, (int)threadIdx.x >> 5, shift, (int)all,
                (int)first, vecs, (per + 31) / 32 * 32};
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
  r.scale = 1.4426950408889634074 / (double)temp;
  if (tid < 256) sm.table[tid] = exp2((double)tid / 256.0 + (double)a.q);
  if (tid == ST - 1) {
    sm.n_cand = 0;
    sm.first = LAST;
    sm.off_min = log2((double)min_p) / r.scale;  // w >= min_p where x >= top + this
    sm.off_low = (a.q + 2.0) / r.scale;          // what is further below rounds to nothing
  }
  for (int i = tid; i < 2 * BINS; i += ST) sm.hist[0][i] = 0;
  asm volatile("cp.async.wait_group 0;" ::: "memory");
  __syncthreads();

  // ---- 1: the largest
  {
    float best = -CUDART_INF_F;
    r.each4([&](const float *x, int) { best = fmaxf(fmaxf(best, fmaxf(x[0], x[1])), fmaxf(x[2], x[3])); });
    const uint32_t k = __reduce_max_sync(0xffffffffu, key_of(best));
    if (lane == 0) sm.warp2[warp] = k;
    __syncthreads();
    if (warp == 0) {
      const uint32_t v = __reduce_max_sync(0xffffffffu, lane < SW ? sm.warp2[lane] : 0);
      if (lane == 0) sm.x[0] = v;
    }
    r.sync();
    r.top = of_key(__reduce_max_sync(0xffffffffu, lane < a.cluster ? (uint32_t)peer64(&sm.x[0], lane) : 0));
  }
  const bool empty = r.top == -CUDART_INF_F;
  if (empty || !(temp > 0.0f) || top_k == 1 || top_p <= 0.0f || min_p > 1.0f) {  // (the same for the whole cluster)
    uint32_t at = LAST;
    if (!empty)
      r.each([&](float x, int i) {
        if (x == r.top) at = min(at, (uint32_t)i);
      });
    at = __reduce_min_sync(0xffffffffu, at);
    if (lane == 0) atomicMin(&sm.first, at);
    r.sync();
    if (rank == 0 && warp == 0) {
      at = __reduce_min_sync(0xffffffffu, lane < a.cluster ? peer32(&sm.first, lane) : (uint32_t)LAST);
      if (lane == 0) {
        a.p.tok[row] = empty ? -1 : (int)at;
        if (a.p.prob) a.p.prob[row] = empty ? 0.0f : 1.0f;
        if (a.p.kept) a.p.kept[row] = empty ? 0 : 1;
      }
    }
    r.sync();  // (others may be reading what this CTA told)
    return;
  }
  const bool inf = r.top == CUDART_INF_F;
  r.cx = -MAXF;
  if (min_p > 0.0f) r.cx = inf ? r.top : fminf(fmaxf(__double2float_ru((double)r.top + sm.off_min), -MAXF), r.top);
  r.low = inf ? r.top : fmaxf(__double2float_rd((double)r.top - sm.off_low), -MAXF);
  // steps of 2^(1/256): of the logits themselves where they keep 2^-40 of one
  // (the last bits of what is below 2^-126 count at temperatures like 2^-80 only)
  r.step = 256.0 * r.scale;
  r.zero = 6755399441055744.0;
  r.exact = inf || temp < 0x1p-80f || !(fabs((double)r.top * r.step) < 0x1p50);
  if (r.exact) r.step = 256.0;
  else r.zero -= rint((double)r.top * r.step);

  // ---- 2, 3: the cut of top-k, then of top-p
  bool do_k = top_k > 0 && top_k < a.n, do_p = top_p < 1.0f;
  const float per_unit = fmaxf(fminf(16.0f / temp, 1e30f), 1e-38f);  // (not 0, which times infinity is NaN)
  // y in bins
  auto place = [&](float x) { return x == r.top ? 0.0f : (r.top - x) * per_unit; };
  bool added = false;   // sum and n have what is before the tokens in question
  float from_bin = 0.0f;  // where those begin
  u64 sum = 0;
  uint32_t n = 0;
  for (bool again = false; do_k || do_p; again = true) {
    const bool weigh = !do_k;  // top-p of all that is kept: their exact weight
    if (again) {
      r.sync();  // (the histogram has been read)
      for (int i = tid; i < 2 * BINS; i += ST) sm.hist[0][i] = 0;
      if (tid == 0) sm.n_cand = 0;
      __syncthreads();
    }
    uint32_t *hist = sm.hist[lane & 1];
    u64 weight = 0;
    if (weigh) {
      r.each4([&](const float *x, int i) {
        weight += r.sum_kept(x, i);
#pragma unroll
        for (int e = 0; e < 4; e++) {
          if (!r.kept(x[e], i + e)) continue;
          const float d = place(x[e]);
          if (d < (float)(BINS - 1)) {  // 2^((b + 1 - d) / 16 nat) of the bin's lowest weight
            const int b = (int)d;
            float over;
            asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(over) : "f"(((float)(b + 1) - d) * (1.4426950408889634f / 16.0f)));
            atomicAdd(hist + b, (uint32_t)__float2int_rn(over * a.unit));
          }
        }
      });
      r.sum_to(weight, 1);
    } else {
      r.each([&](float x, int i) {
        if (r.kept(x, i)) atomicAdd(hist + (int)fminf(place(x), (float)(BINS - 1)), 1u);  // (NaN, of infinities: the last)
      });
    }
    __syncthreads();
    sm.hist[0][tid] += sm.hist[1][tid];
    if (tid == 0) sm.lo = sm.hi = BINS - 1;
    r.sync();
    if (weigh) weight = r.all_sum(1);
    // bin tid of the whole row, and the sums down to it: tokens (for top-p, what
    // they are at the most), weights
    uint32_t c = 0;
    float m = 0.0f;
    {
      uint32_t v[8];
#pragma unroll
      for (int k = 0; k < 8; k++) v[k] = k < a.cluster ? peer32(&sm.hist[0][tid], k) : 0;
#pragma unroll
      for (int k = 0; k < 8; k++) {
        m += (float)v[k];
        c += !weigh ? v[k] : v[k] ? (uint32_t)((float)v[k] * (1.0f / a.unit)) + 1 : 0;
      }
      m *= exp2f((float)(tid + 1) * (-1.4426950408889634f / 16.0f));
      if (weigh && tid == BINS - 1) c = (uint32_t)a.n;  // (not counted)
    }
    uint32_t cs = c;
    float ms = m;
#pragma unroll
    for (int i = 1; i < 32; i *= 2) {
      const uint32_t y = __shfl_up_sync(0xffffffffu, cs, i);
      const float z = __shfl_up_sync(0xffffffffu, ms, i);
      if (lane >= i) cs += y, ms += z;
    }
    if (lane == 31) sm.warp2[warp] = cs, sm.warpf[warp] = ms;
    __syncthreads();
    uint32_t total = 0, cb = 0;
    float mass = 0.0f, mb = 0.0f;
#pragma unroll
    for (int w = 0; w < SW; w++) {
      if (w == warp) cb = total, mb = mass;
      total += sm.warp2[w];
      mass += sm.warpf[w];
    }
    cs += cb, ms += mb;
    const uint32_t k = min((uint32_t)top_k, total);
    // (sums of weights need not ascend by the last bit: the first bin that passes)
    uint32_t l = BINS - 1, h = BINS - 1;
    if (do_k ? cs >= k : ms >= mass * top_p * (1.0f - a.margin)) l = tid;
    if (do_k ? cs >= k : ms >= mass * top_p * (1.0f + a.margin)) h = tid;
    l = __reduce_min_sync(0xffffffffu, l);
    h = __reduce_min_sync(0xffffffffu, h);
    if (lane == 0 && l < BINS - 1) atomicMin(&sm.lo, l);
    if (lane == 0 && h < BINS - 1) atomicMin(&sm.hi, h);
    __syncthreads();
    const int hi = (int)sm.hi;
    int lo = (int)sm.lo;
    if (tid == hi) sm.at = cs;
    if (tid == lo) sm.above = cs - c;
    __syncthreads();
    const uint32_t down = sm.at;  // tokens down to bin hi
    uint32_t above = sm.above;    // before bin lo
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
    const float d_lo = (float)lo, d_hi = hi == BINS - 1 ? CUDART_INF_F : (float)(hi + 1);
    auto side = [&](float x, int i) {  // 0: in question, 1: before, -1: behind
      if (by_order) {
        const u64 o = order_of(x, i);
        return o > o_hi ? 1 : o < o_lo ? -1 : 0;
      }
      const float d = place(x);
      return d < d_lo ? 1 : d >= d_hi && hi < BINS - 1 ? -1 : 0;
    };
    const double target = (double)top_p * (double)weight;
    if (inside > CAP) {
      // Halving.  The order's bounds first, and the exact weight before them.
      u64 least = ~0ull, most = 0, before = 0, n_in = 0;
      r.each([&](float x, int i) {
        if (!r.kept(x, i)) return;
        const int s = side(x, i);
        if (s == 0) n_in++, least = min(least, order_of(x, i)), most = max(most, order_of(x, i));
        if (s > 0 && weigh) before += r.fixed(x);
      });
#pragma unroll
      for (int j = 16; j > 0; j >>= 1) least = min(least, __shfl_xor_sync(0xffffffffu, least, j)), most = max(most, __shfl_xor_sync(0xffffffffu, most, j));
      __syncthreads();
      r.sum_to(before, 2);
      __syncthreads();
      r.sum_to(n_in, 5);
      __syncthreads();
      if (tid == 0) sm.x[3] = ~0ull, sm.x[4] = 0;
      __syncthreads();
      if (lane == 0) atomicMin(&sm.x[3], least), atomicMax(&sm.x[4], most);
      r.sync();
      base_w = r.all_sum(2);
      inside = (uint32_t)r.all_sum(5);
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
    added = weigh && !by_order;
    from_bin = d_lo;
    sum = 0;
    n = 0;
    const uint32_t to = map_rank(shaddr(&sm.cand[0]), 0), counter = map_rank(shaddr(&sm.n_cand), 0);
    r.each4([&](const float *x, int i) {
      bool before[4];
#pragma unroll
      for (int e = 0; e < 4; e++) {
        const bool on = r.kept(x[e], i + e);
        const int s = on ? side(x[e], i + e) : -1;
        before[e] = s > 0 && x[e] >= r.low;
        n += s > 0;
        if (s == 0) {
          uint32_t at;
          asm volatile("atom.relaxed.cluster.shared::cluster.add.u32 %0, [%1], 1;" : "=r"(at) : "r"(counter) : "memory");
          if (at < CAP) asm volatile("st.shared::cluster.u64 [%0], %1;" ::"r"(to + at * 8), "l"(order_of(x[e], i + e)) : "memory");
        }
      }
      if (added) r.add4(x, before, sum);
    });
    if (added) r.sum_to(sum, 5);
    r.sync();
    if (rank == 0) {
      if (added) base_w = r.all_sum(5);
      const int nc = min((int)sm.n_cand, CAP);
      u64 v = tid < nc ? sm.cand[tid] : 0;
      int n2 = 32;
      while (n2 < nc) n2 *= 2;
      __syncthreads();
      if (warp * 32 < n2) {  // (whole warps; the barrier below is theirs)
        for (int size = 2; size <= n2; size *= 2)
          for (int j = size / 2; j > 0; j /= 2) {
            u64 o;
            if (j >= 32) {
              sm.cand[tid] = v;
              asm volatile("bar.sync 1, %0;" ::"r"(n2) : "memory");
              o = sm.cand[tid ^ j];
              asm volatile("bar.sync 1, %0;" ::"r"(n2) : "memory");
            } else {
              o = __shfl_xor_sync(0xffffffffu, v, j);
            }
            const bool down_here = (tid & size) == 0, low_half = (tid & j) == 0;
            v = down_here == low_half ? max(v, o) : min(v, o);
          }
      }
      const float x = of_key((uint32_t)(v >> 32));
      // the last one that top-k leaves
      const int most = do_k ? min(nc, (int)(k - above)) : nc;
      int cut = most - 1;
      if (!do_k || both) {
        const u64 w = tid < most ? r.fixed(x) : 0, b = r.scan(w);
        double goal = target;
        if (both) {
          if (tid == ST - 1) sm.x[4] = b + w;
          __syncthreads();
          goal = (double)top_p * (double)sm.x[4];
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

  // ---- 4: the kept weights by index (of what came before the tokens in question they are there)
  if (!added) sum = 0, n = 0;
  r.each4([&](const float *x, int i) {
    const float least = fmaxf(r.cx, r.low);
    bool on[4];
#pragma unroll
    for (int e = 0; e < 4; e++) {
      on[e] = r.kept(x[e], i + e) && !(added && place(x[e]) < from_bin);
      n += on[e];
      on[e] = on[e] && x[e] >= least;
    }
    r.add4(x, on, sum);
  });
  sum = r.sum_warp(sum);
  n = __reduce_add_sync(0xffffffffu, n);
  __syncthreads();  // (sums of before have been read)
  if (lane == 0) sm.warp[warp] = sum, sm.warp2[warp] = n;
  __syncthreads();
  if (warp == 0) {
    const u64 w = r.sum_warp(lane < SW ? sm.warp[lane] : 0);
    const uint32_t c = __reduce_add_sync(0xffffffffu, lane < SW ? sm.warp2[lane] : 0);
    if (lane == 0) sm.x[2] = w, sm.x[3] = c;  // (another CTA may still read x[0])
  }
  r.sync();
  u64 all_w = 0, before = 0, all_n = 0;
  {
    u64 w[8], c[8];
#pragma unroll
    for (int j = 0; j < 8; j++) {
      w[j] = j < a.cluster ? peer64(&sm.x[2], j) : 0;
      c[j] = j < a.cluster ? peer64(&sm.x[3], j) : 0;
    }
#pragma unroll
    for (int j = 0; j < 8; j++) {
      if (j < rank) before += w[j];
      all_w += w[j];
      all_n += c[j];
    }
  }
  // the first token whose sum passes floor(u W) passes u W (u below 0 and NaN: the first)
  const double goal = (double)u * (double)all_w;
  u64 pass = goal > 0.0 ? (goal < 9.2e18 ? (u64)goal : all_w) : 0;
  pass = min(pass, all_w - 1);
  if (pass >= before && pass - before < sm.x[2]) {  // one CTA: of the warp in whose run it falls all threads take a vector
    u64 from = before;
    int w = 0;
    while (w < SW - 1 && pass >= from + sm.warp[w]) from += sm.warp[w++];
    __syncthreads();
    const int w1 = min(vecs, (w + 1) * r.per);
    for (int i0 = w * r.per; i0 < w1; i0 += ST) {
      float x[V];
      const int i = i0 + tid, token = r.p0 + i * V - shift;
      u64 mine = 0;
      if (i < w1) {
        r.vec(i, x);
#pragma unroll
        for (int e = 0; e < V; e += 4) mine += r.sum_kept(x + e, token + e);
      }
      const u64 b0 = from + r.scan(mine);
      if (mine && pass >= b0 && pass < b0 + mine) {
        u64 b = b0;
#pragma unroll
        for (int e = 0; e < V; e++) {
          const u64 one = r.kept(x[e], token + e) ? r.fixed(x[e]) : 0;
          if (pass >= b && pass < b + one) {
            a.p.tok[row] = token + e;
            if (a.p.prob) a.p.prob[row] = (float)(r.weight(x[e]) / (double)all_w);
            if (a.p.kept) a.p.kept[row] = (int)all_n;
          }
          b += one;
        }
      }
      if (i0 + ST < w1) {  // (runs longer than the threads)
        if (tid == ST - 1) sm.x[4] = b0 + mine;
        __syncthreads();
        from = sm.x[4];
        __syncthreads();
      }
    }
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
  // CTAs a row: by what they hold, two an SM, one where rows are longer; more where the rows leave SMs without any
  const long long vecs = ((long long)n + 2 * v - 2) / v, most = 96 * 1024 / 16, wide = 208 * 1024 / 16;
  long long c = std::min(8LL, (vecs + most - 1) / most);
  while (c < 8 && rows * c * 2 <= 148 && vecs >= 512 * c) c *= 2;
  c = std::min(c, 8LL);
  const long long seg = (vecs + c - 1) / c;
  const bool big = seg > wide;
  a.cluster = (int)c;
  a.seg = (int)(seg * v);
  // a weight is at most 1.0645 of its bin's lowest: in 2^-15 steps 65536 of a bin and CTA fit 32 bits
  a.unit = 32768.0f;
  for (long long x = 65536; x < a.seg; x *= 2) a.unit *= 0.5f;
  a.margin = MARGIN + 1.0f / a.unit;
  const int smem = (int)sizeof(Smem) + (big ? 0 : (int)(seg * 16));
  const dim3 grid((unsigned)(rows * c)), block(ST);
#define GO(E) launch_cluster(big ? k_sample<E, true> : k_sample<E, false>, (int)c, grid, block, smem, st, a)
  return type == T_F32 ? GO(float) : type == T_F16 ? GO(__half) : GO(__nv_bfloat16);
#undef GO
}

}  // namespace pk
