// pk_sample.cu -- a token for every row of logits, from given random numbers
// (pk_sample_rows): temperature, min-p, top-k and top-p.  pk_sample takes one
// row in the reference's order of operations (sampler.rs:21-92), with its sort.
//
//   w_t = 2^(y_t), y_t = (x_t - max x) log2(e) / temp;  order: x down, index up
// All three rules keep a beginning of that order, so what is kept is everything
// down to one (logit, index), the cut.  Without a sort of the row:
//   1  the largest logit: y <= 0.  min_p is a least logit.
//   2  a histogram: for top-k of y, for top-p of the weights by their exponents
//      and first three bits, in 2^-15 of the exponent's power (a 6e-5th is
//      allowed for that).  Its sums from the top say which bins hold the cut, and
//      a search among floats, by the same function, which logits begin and end
//      them.
//   3  the tokens of those bins (or of all bins down to there, if they are few,
//      for top-k and top-p at once) are sorted by one CTA and added up exactly,
//      beginning with the exact weight above them.  If they are too many, as in rows of equal logits,
//      halving steps on (logit, index) come before.
//   4  sums of the kept weights by index, the token in whose part u falls.
// A token depends on sums of a whole vocabulary next to whose borders u may lie:
// at 128256 borders an error of 2^-24 would change one token in a hundred.  So
// weights are made in double, 2^y from a table and a few terms of the series
// (1.4e-13), and added as 64-bit integers, in which no order matters: 2^-q steps
// of the largest, n 2^q <= 2^62.
//
// A row is read once, into the shared memory of a cluster of up to 8 CTAs, and
// gone over there; rows that do not fit are read again each time.
#include <math_constants.h>

#include <algorithm>
#include <type_traits>

#include "pk_cache.cuh"
#include "pk_cache.h"
#include "pk_launch.h"

namespace pk {
namespace {

typedef unsigned long long u64;

constexpr int ST = 512, SW = ST / 32;  // threads, warps
constexpr int BINS = 512, CAP = 512;   // of the histogram; tokens that one CTA sorts
static_assert(BINS == ST && CAP == ST, "a bin and a sorted token a thread");
constexpr int TB = 4, TABLE = 1 << TB;  // table of 2^(i / TABLE): 16 entries of 8 bytes are in different banks
constexpr float MARGIN = 6e-5f;        // of sums of the histogram's weights, with 16 bits of each
constexpr int LAST = 0x7fffffff;
constexpr float MAXF = 3.402823466e38f;

struct SampleK {
  const void *logits;
  long long stride;
  int n, cluster, seg;   // seg: positions a CTA, whole 16-byte vectors
  int q;                 // fixed-point bits of a weight
  int drop;              // bits of a weight's 21 that the histogram leaves out
  pk_sample_args p;
};

struct Smem {  // behind the row's values
  uint32_t hist[2][BINS];  // of even and of odd lanes, which then collide less
  u64 cand[CAP];
  double table[TABLE];
  u64 warp[SW], x[6];   // of the CTA's warps; what the cluster's CTAs tell each other
  double off_min, off_low;
  uint32_t warp2[SW], n_cand, lo, hi, at, above, first;
  float warpf[SW], cut_x, edge[2];
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
  float top = 0.0f, low = 0.0f, none = 0.0f;  // the largest logit; what is below `low` has no weight, nor has `none`
  double step = 0.0, zero = 0.0;  // TABLE log2(e) / temp; 1.5 * 2^52 less the largest logit's steps
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
  __device__ __forceinline__ void kept4(const float *x, int i, bool (&on)[4]) const {
#pragma unroll
    for (int e = 0; e < 4; e++) on[e] = x[e] >= cx;
    if (ci != LAST) {
#pragma unroll
      for (int e = 0; e < 4; e++) on[e] = on[e] && (x[e] > cx || i + e <= ci);
    }
  }

  // The weight times 2^q (and a factor within 2^(1/2/TABLE) of 1, the same for
  // the whole row), for x <= top; EX: as `exact` says.  What is below `low`, and
  // `none`, have one that rounds to 0: without EX x has to be `none` or more.
  template <bool EX>
  __device__ __forceinline__ double weight_as(float x) const {
    double v;
    if (EX) {
      v = x == top ? 0.0 : x >= low ? ((double)x - (double)top) * scale : -100.0;
    } else {  // x in double without the conversion, of which an SM makes 16 a cycle; 0 and subnormals become up to 2^-126
      const int u = __float_as_int(x);
      v = __hiloint2double(((u >> 3) & 0x8fffffff) + (896 << 20), u << 29);
    }
    const double t = fma(v, step, zero);  // its low bits are the number of steps, rounded
    const double r = fma(v, step, zero - t);  // what is left of them, -0.5 .. 0.5
    const int k = __double2loint(t);
    // 2^(r / TABLE): terms (ln(2) / TABLE)^i / i!
    constexpr double L = 0.6931471805599453 / TABLE;
    double f = fma(L * L * L * L * L / 120, r, L * L * L * L / 24);
    f = fma(f, r, L * L * L / 6);
    f = fma(f, r, L * L / 2);
    f = fma(f, r, L);
    f = fma(f, r, 1.0) * sm.table[k & (TABLE - 1)];
    return __hiloint2double(__double2hiint(f) + ((k & ~(TABLE - 1)) << (20 - TB)), __double2loint(f));
  }
  __device__ __forceinline__ double weight(float x) const {
    x = fmaxf(x, none);
    return exact ? weight_as<true>(x) : weight_as<false>(x);
  }
  // the same, rounded to an integer, plus ONE
  static constexpr u64 ONE = 0x4330000000000000ull;  // 2^52's bits
  __device__ __forceinline__ u64 raw(double w) const { return (u64)__double_as_longlong(w + 4503599627370496.0); }
  __device__ __forceinline__ u64 fixed(float x) const { return raw(weight(x)) - ONE; }
  // f(std::true_type or std::false_type), as `exact` is: passes that make weights, twice in the code
  template <class F>
  __device__ __forceinline__ void as_exact(F f) const {
    if (exact) f(std::true_type{});
    else f(std::false_type{});
  }
  // of four those that are `on`
  template <bool EX>
  __device__ __forceinline__ void add4(const float *x, const bool (&on)[4], u64 &sum) const {
    if (!(on[0] || on[1] || on[2] || on[3])) return;
#pragma unroll
    for (int e = 0; e < 4; e++) sum += raw(weight_as<EX>(on[e] ? fmaxf(x[e], none) : none)) - ONE;
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
  if (tid < TABLE) sm.table[tid] = exp2((double)tid / TABLE + (double)a.q);
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
  // steps of 2^(1/TABLE): of the logits themselves where they keep 2^-40 of one
  // (the last bits of what is below 2^-126 count at temperatures like 2^-80 only)
  r.step = TABLE * r.scale;
  r.zero = 6755399441055744.0;
  r.none = r.low;
  r.exact = inf || temp < 0x1p-80f || !(fabs((double)r.top * r.step) < 0x1p50) || !(r.low > -MAXF);
  if (r.exact) r.step = TABLE, r.none = -CUDART_INF_F;
  else r.zero -= rint((double)r.top * r.step);

  // ---- 2, 3: the cut of top-k, then of top-p
  bool do_k = top_k > 0 && top_k < a.n, do_p = top_p < 1.0f;
  // bins of 1/16 nat for top-k: to the nearest, by an addition in which the
  // sum's last bits are the number (what the constant loses shifts all alike)
  const float per_unit = fmaxf(fminf(16.0f / temp, 1e30f), 1e-38f);
  const float bias = fminf(fmaxf(rintf(r.top * per_unit), -4e6f), 4e6f);
  const bool near = fabsf(r.top * per_unit) < 4e6f;
  auto bin_k = [&](float x) {
    const float d = near ? fmaf(x, -per_unit, bias) : x == r.top ? 0.0f : (r.top - x) * per_unit;
    return __float_as_uint(fminf(fmaxf(d, 0.0f), (float)(BINS - 1)) + 8388608.0f) & 1023u;  // (NaN, of infinities: 0)
  };
  // for top-p by the weight's exponent and three bits: bin 0 has the largest
  const int hi_top = __double2hiint(r.weight(r.top)) >> 17;
  auto bin_p = [&](double w) { return (uint32_t)min(hi_top - (__double2hiint(w) >> 17), BINS - 1); };
  float before_x = CUDART_NAN_F;  // logits from here on are before those in question
  bool added = false;             // sum and n have them
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
      r.as_exact([&](auto ex) {
        r.each4([&](const float *x, int i) {
          bool on[4];
          r.kept4(x, i, on);
#pragma unroll
          for (int e = 0; e < 4; e++) {
            const double w = r.template weight_as<decltype(ex)::value>(on[e] ? fmaxf(x[e], r.none) : r.none);
            weight += r.raw(w) - r.ONE;
            if (on[e] && x[e] >= r.low) atomicAdd(hist + bin_p(w), ((__double2hiint(w) & 0xfffffu) | 0x100000u) >> a.drop);
          }
        });
      });
      weight = r.sum_warp(weight);
      if (lane == 0) sm.warp[warp] = weight;
    } else {
      r.each4([&](const float *x, int i) {
        bool on[4];
        r.kept4(x, i, on);
#pragma unroll
        for (int e = 0; e < 4; e++)
          if (on[e]) atomicAdd(hist + bin_k(x[e]), 1u);
      });
    }
    __syncthreads();
    sm.hist[0][tid] += sm.hist[1][tid];
    if (weigh && warp == 0) {
      weight = r.sum_warp(lane < SW ? sm.warp[lane] : 0);
      if (lane == 0) sm.x[1] = weight;
    }
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
        c += weigh ? v[k] >> (20 - a.drop) : v[k];
      }
      m *= exp2f((float)(((hi_top - tid) >> 3) - (hi_top >> 3)));
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
    if (do_k ? cs >= k : ms >= mass * top_p * (1.0f - MARGIN)) l = tid;
    if (do_k ? cs >= k : ms >= mass * top_p * (1.0f + MARGIN)) h = tid;
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
    // The least floats of bins below lo (that are before those in question) and
    // of bins up to hi, a warp each: 33 floats around where the bin should end,
    // or, if it does not there, 33 that divide all, and so on.
    if (warp < 2) {
      const int b = warp == 0 ? lo - 1 : hi;
      auto in = [&](uint32_t key) {
        const float x = of_key(key);
        return (int)(do_k ? bin_k(x) : x >= r.low ? bin_p(r.weight(x)) : (uint32_t)(BINS - 1)) <= b;
      };
      const uint32_t least = key_of(-CUDART_INF_F);
      uint32_t from = least, to = key_of(r.top);  // (of which one is not looked at, the other is in bin 0)
      if (b < 0 || b == BINS - 1) {
        from = to = b < 0 ? 0 : key_of(-MAXF);
      } else {
        double g;
        if (do_k) g = ((double)bias - b - 0.5) / (double)per_unit;
        else g = (log2(__hiloint2double((hi_top - b) << 17, 0)) - a.q) * TABLE;
        if (!do_k) g = r.exact ? (double)r.top + g / TABLE / r.scale : (g - (r.zero - 6755399441055744.0)) / r.step;
        const uint32_t at = min(max(key_of((float)g), least + 17), to - min(to - least - 17, 16u));
        const bool here = lane == 0 ? !in(at - 16) : lane == 1 ? in(at + 16) : true;
        if (to - least > 64 && __all_sync(0xffffffffu, here)) from = at - 16, to = at + 16;
      }
      while (to - from > 1) {
        const uint32_t step = (to - from + 31) / 32, at = from + min((uint32_t)(lane + 1) * step, to - from);
        const uint32_t lanes = __ballot_sync(0xffffffffu, in(at));  // (`to` is among them)
        const int f = __ffs(lanes) - 1;
        const uint32_t next = __shfl_sync(0xffffffffu, at, f);
        from = f > 0 ? __shfl_sync(0xffffffffu, at, max(f - 1, 0)) : from;
        to = next;
      }
      if (lane == 0) sm.edge[warp] = b < 0 ? CUDART_NAN_F : of_key(to);
    }
    __syncthreads();
    before_x = sm.edge[0];
    const float last_x = weigh ? fmaxf(sm.edge[1], r.low) : sm.edge[1];  // (what has no weight is not in the histogram)
    // (by logits, or after halving by order) is it in question? is it before?
    u64 o_lo = 0, o_hi = ~0ull, base_w = 0;
    bool by_order = false;
    auto side = [&](float x, int i) {  // 0: in question, 1: before, -1: behind
      if (by_order) {
        const u64 o = order_of(x, i);
        return o > o_hi ? 1 : o < o_lo ? -1 : 0;
      }
      return x >= before_x ? 1 : x >= last_x ? 0 : -1;
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
    sum = 0;
    n = 0;
    const uint32_t to = map_rank(shaddr(&sm.cand[0]), 0), counter = map_rank(shaddr(&sm.n_cand), 0);
    auto take = [&](float x, int i) {
      uint32_t at;
      asm volatile("atom.relaxed.cluster.shared::cluster.add.u32 %0, [%1], 1;" : "=r"(at) : "r"(counter) : "memory");
      if (at < CAP) asm volatile("st.shared::cluster.u64 [%0], %1;" ::"r"(to + at * 8), "l"(order_of(x, i)) : "memory");
    };
    if (by_order) {
      r.each([&](float x, int i) {
        if (r.kept(x, i) && side(x, i) == 0) take(x, i);
      });
    } else {
      r.as_exact([&](auto ex) {
        r.each4([&](const float *x, int i) {
          if (!(x[0] >= last_x || x[1] >= last_x || x[2] >= last_x || x[3] >= last_x)) return;
          bool on[4], before[4];
          r.kept4(x, i, on);
#pragma unroll
          for (int e = 0; e < 4; e++) {
            before[e] = on[e] && x[e] >= before_x;
            n += before[e];
            if (on[e] && !before[e] && x[e] >= last_x) take(x[e], i + e);
          }
          if (added) r.template add4<decltype(ex)::value>(x, before, sum);
        });
      });
      if (added) r.sum_to(sum, 5);
    }
    r.sync();
    u64 *sorted = reinterpret_cast<u64 *>(sm.hist[0]);  // (which has been read)
    static_assert(sizeof(sm.hist) >= CAP * sizeof(u64), "room");
    if (rank == 0) {
      if (added) base_w = r.all_sum(5);
      const int nc = min((int)sm.n_cand, CAP), lists = (nc + 31) / 32;
      u64 v = tid < nc ? sm.cand[tid] : 0;
      __syncthreads();
      if (warp < lists) {  // each warp sorts its 32
#pragma unroll
        for (int size = 2; size <= 32; size *= 2)
#pragma unroll
          for (int j = size / 2; j > 0; j /= 2) {
            const u64 o = __shfl_xor_sync(0xffffffffu, v, j);
            const bool down_here = (lane & size) == 0, low_half = (lane & j) == 0;
            v = down_here == low_half ? max(v, o) : min(v, o);
          }
        sm.cand[tid] = v;
      }
      __syncthreads();
      if (warp < lists) {  // and finds how many of the other lists' are before each
        int place = lane;
#pragma unroll 4
        for (int w = 0; w < lists; w++) {
          const u64 *o = sm.cand + 32 * w;
          int b = 0;
#pragma unroll
          for (int j = 16; j > 0; j /= 2) b += o[b + j - 1] > v ? j : 0;
          b += o[b] > v;
          place += w == warp ? 0 : b;
        }
        __syncwarp();
        if (v) sorted[place] = v;
      }
      __syncthreads();
      v = tid < nc ? sorted[tid] : 0;
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
  if (!added) sum = 0, n = 0, before_x = CUDART_NAN_F;
  r.as_exact([&](auto ex) {
    if (r.ci == LAST && r.cx <= r.none) {  // nothing is cut off that has a weight
      uint32_t made = 0;
      r.each4([&](const float *x, int) {
#pragma unroll
        for (int e = 0; e < 4; e++) {
          n += x[e] >= r.cx;
          sum += r.raw(r.template weight_as<decltype(ex)::value>(fmaxf(x[e], r.none)));
        }
        made += 4;
      });
      sum -= made * r.ONE;
    } else {
      r.each4([&](const float *x, int i) {
        if (!(x[0] >= r.cx || x[1] >= r.cx || x[2] >= r.cx || x[3] >= r.cx)) return;
        bool on[4];
        r.kept4(x, i, on);
#pragma unroll
        for (int e = 0; e < 4; e++) {
          on[e] = on[e] && !(x[e] >= before_x);
          n += on[e];
        }
        r.template add4<decltype(ex)::value>(x, on, sum);
      });
    }
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
        for (int e = 0; e < V; e++) mine += r.kept(x[e], token + e) ? r.fixed(x[e]) : 0;
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
  while (c < 8 && rows * c * 2 <= 296 && vecs >= 512 * c) c *= 2;
  c = std::min(c, 8LL);
  const long long seg = (vecs + c - 1) / c;
  const bool big = seg > wide;
  a.cluster = (int)c;
  a.seg = (int)(seg * v);
  // 21 bits of a weight, of which 16 are kept: 65536 of a bin and CTA fit 32 bits
  a.drop = 5;
  for (long long x = 65536; x < a.seg; x *= 2) a.drop++;
  const int smem = (int)sizeof(Smem) + (big ? 0 : (int)(seg * 16));
  const dim3 grid((unsigned)(rows * c)), block(ST);
#define GO(E) launch_cluster(big ? k_sample<E, true> : k_sample<E, false>, (int)c, grid, block, smem, st, a)
  return type == T_F32 ? GO(float) : type == T_F16 ? GO(__half) : GO(__nv_bfloat16);
#undef GO
}

}  // namespace pk
