// pk_sample.cu -- a token for every row of logits, from given random numbers
// (pk_sample_rows): temperature, min-p, top-k and top-p.  pk_sample takes one
// row in the reference's order of operations (sampler.rs:21-92), with its sort.
//
//   w_t = 2^(y_t), y_t = (x_t - max x) log2(e) / temp;  order: x down, index up
// All three rules keep a beginning of that order, so what is kept is everything
// down to one (logit, index), the cut.  Without a sort of the row:
//   1  the largest logit: y <= 0.  min_p is a least logit.
//   2  a histogram.  For top-k of the threads' largest logits by y: the k-th of
//      them is a lower bound of the k-th of all that few more logits pass.  Where
//      k is too large for that, of all logits.  For top-p of all weights, made in
//      f32, by their exponents and first five bits, in 2^-15 of the exponent's
//      power (a 6e-5th is allowed for all that).  Its sums from the top say which
//      bins hold the cut, and a search among floats, by the same function, which
//      logits begin and end them.
//   3  one pass makes the exact sums of all weights and of those before the bins
//      in question, and collects these bins' tokens in one CTA, which sorts them
//      and adds them up.  If they are too many, as in rows of equal logits, exact
//      histograms of 512 parts of the order come before.  Where nothing is before them, as for
//      top-k, that CTA has all it needs for top-p and the token, too.
//   4  else sums of the kept weights by index, the token in whose part u falls.
// A token depends on sums of a whole vocabulary next to whose borders u may lie:
// at 128256 borders an error of 2^-24 would change one token in a hundred.  So
// weights are made in double, 2^y from a table and a few terms of the series
// (1.4e-13), and added as 64-bit integers, in which no order matters: 2^-q steps
// of the largest, n 2^q <= 2^62.
//
// A row is read once, into the shared memory of a cluster of up to 8 CTAs, and
// gone over there; rows that do not fit are read again each time.
//
// Measured: 250 f32 rows of 128256: the largest alone 45 us, temperature alone
// 90, top-k 40 88, top-p 0.6 at temperature 1.5 209, rows with rules of their own
// 141 to 156 by the rows (their bytes take 20); 64 bf16 rows of 73448, top-p 0.9:
// 41; one f32 row of 73448, all rules: 10.  What bounds it: instructions (60 M for
// the 250 rows with rules, 1.8 a cycle and SM; 33 an element for an exact weight)
// and the steps that a cluster takes one after another, during which two CTAs an SM
// leave it half idle.  With rules 348 (f32) or 532 bytes a thread spill at the 64
// registers that two CTAs an SM allow, 596 and 1,440 where rows are read again.
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
constexpr int BINS = 1024, CAP = 512;  // of the histogram; tokens that one CTA sorts
constexpr int FEW = 128;               // that one warp sorts
static_assert(BINS == 2 * ST && CAP == ST, "two bins and a sorted token a thread");
constexpr int TB = 4, TABLE = 1 << TB;  // table of 2^(i / TABLE): 16 entries of 8 bytes are in different banks
constexpr float MARGIN = 3e-5f;        // of the histogram's weights in f32, besides the bits that they lose
constexpr int LAST = 0x7fffffff;
constexpr float MAXF = 3.402823466e38f;

struct SampleK {
  const void *logits;
  long long stride;
  int n, cluster, seg;   // seg: positions a CTA, whole 16-byte vectors
  int q;                 // fixed-point bits of a weight
  int drop;              // bits of a weight's 24 that the histogram leaves out
  float margin;          // what its sums may be off by
  pk_sample_args p;
};

struct Smem {  // behind the row's values
  uint32_t hist[2][BINS];  // of even and of odd lanes, which then collide less
  u64 cand[CAP];
  double table[TABLE];
  u64 warp[SW], warpb[SW], told[2], x[6];   // of the CTA's warps; what the cluster's CTAs tell each other
  double off_min, off_low;
  u64 base_w;
  uint32_t warp2[SW], n_cand, lo, hi, at, above, inside, first;
  float warpf[SW], cut_x, edge[2];
  uint32_t n_all;
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

// Lane l holds elements l, 32 + l ..: sorted, the largest first.
template <int J>
__device__ __forceinline__ void sort_warp(u64 (&v)[J], int lane) {
#pragma unroll
  for (int size = 2; size <= 32 * J; size *= 2)
#pragma unroll
    for (int j = size / 2; j > 0; j /= 2)
#pragma unroll
      for (int i = 0; i < J; i++) {
        const bool down = ((i * 32 + (size < 32 ? lane : 0)) & size) == 0;
        const bool falls = size < 32 ? (lane & size) == 0 : down;
        if (j >= 32) {
          const int o = i ^ (j / 32);
          if (o > i) {
            const u64 a = v[i], b = v[o];
            v[i] = falls ? max(a, b) : min(a, b);
            v[o] = falls ? min(a, b) : max(a, b);
          }
        } else {
          const u64 o = __shfl_xor_sync(0xffffffffu, v[i], j);
          v[i] = falls == ((lane & j) == 0) ? max(v[i], o) : min(v[i], o);
        }
      }
}
// Inclusive sums in that order.
template <int J>
__device__ __forceinline__ void scan_warp(u64 (&v)[J], int lane) {
  u64 before = 0;
#pragma unroll
  for (int i = 0; i < J; i++) {
#pragma unroll
    for (int j = 1; j < 32; j *= 2) {
      const u64 y = __shfl_up_sync(0xffffffffu, v[i], j);
      if (lane >= j) v[i] += y;
    }
    v[i] += before;
    before = __shfl_sync(0xffffffffu, v[i], 31);
  }
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
  __device__ __forceinline__ uint4 words(int i) const {  // vector i of this CTA
    if (!BIG) return data[i];
    const long long p = (long long)p0 + (long long)i * V;
    if (p >= shift && p + V <= end) return __ldcg(reinterpret_cast<const uint4 *>(base + (p - shift)));
    uint4 w;
    E *v = reinterpret_cast<E *>(&w);
#pragma unroll
    for (int e = 0; e < V; e++) v[e] = load(p + e);
    return w;
  }
  __device__ __forceinline__ void floats(const uint4 &w, float (&x)[V]) const {
    const E *v = reinterpret_cast<const E *>(&w);
#pragma unroll
    for (int e = 0; e < V; e++) x[e] = to_f(v[e]);
  }
  __device__ __forceinline__ void vec(int i, float (&x)[V]) const { floats(words(i), x); }
  // f(four values, the first's token) for this thread's, in order.  NaN compares as false everywhere.
  template <class F>
  __device__ __forceinline__ void each4(F f) const {
    const int w1 = min(vecs, (warp + 1) * per);
    auto one = [&](int i, const uint4 &w) {
      float x[V];
      floats(w, x);
#pragma unroll
      for (int e = 0; e < V; e += 4) f(x + e, p0 + i * V + e - shift);
    };
    int i = warp * per + lane;
    if (BIG) {  // two vectors ahead
      uint4 w[2];
#pragma unroll
      for (int j = 0; j < 2; j++) w[j] = i + 32 * j < w1 ? words(i + 32 * j) : uint4{};
      for (; i < w1; i += 64) {
#pragma unroll
        for (int j = 0; j < 2; j++) {
          const uint4 now = w[j];
          const int next = i + 32 * j + 64;
          if (next < w1) w[j] = words(next);
          if (i + 32 * j < w1) one(i + 32 * j, now);
        }
      }
    } else {
      for (; i < w1; i += 32) one(i, words(i));
    }
  }
  // the same for whole warps, with -inf past the end
  template <class F>
  __device__ __forceinline__ void each_warp(F f) const {
    const int w1 = min(vecs, (warp + 1) * per);
    for (int i0 = warp * per; i0 < w1; i0 += 32) {
      const int i = i0 + lane;
      float x[V];
      if (i < w1) {
        vec(i, x);
      } else {
#pragma unroll
        for (int e = 0; e < V; e++) x[e] = -CUDART_INF_F;
      }
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
      v = x == top ? 0.0 : x >= low ? fmax(((double)x - (double)top) * scale, -100.0) : -100.0;
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
  // The CTA's n values (0 behind them), the largest first.  Each warp sorts its 32
  // and finds how many of the other lists' are before each of them.
  __device__ __forceinline__ u64 sorted(u64 v, int n) const {
    const int lists = (n + 31) / 32;
    u64 *out = reinterpret_cast<u64 *>(sm.hist[0]);  // (which has been read)
    static_assert(sizeof(sm.hist[0]) >= CAP * sizeof(u64), "room");
    __syncthreads();
    if (warp < lists) {
      u64 one[1] = {v};
      sort_warp(one, lane);
      sm.cand[tid] = v = one[0];
    }
    __syncthreads();
    if (warp < lists) {
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
      if (v) out[place] = v;
    }
    __syncthreads();
    return tid < n ? out[tid] : 0;
  }
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

// The first token whose sum passes floor(u W) passes u W (u below 0 and NaN: the first).
__device__ __forceinline__ u64 pass_of(float u, u64 all) {
  const double goal = (double)u * (double)all;
  return min(goal > 0.0 ? (goal < 9.2e18 ? (u64)goal : all) : 0, all - 1);
}

// RULES: min_p, top_k or top_p are given.
template <class E, bool BIG, bool RULES>
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
  const float top_p = RULES && a.p.top_p ? __ldg(a.p.top_p + row) : 1.0f, min_p = RULES && a.p.min_p ? __ldg(a.p.min_p + row) : 0.0f;
  const int top_k = RULES && a.p.top_k ? __ldg(a.p.top_k + row) : 0;
  r.scale = 1.4426950408889634074 / (double)temp;
  if (tid < TABLE) sm.table[tid] = exp2((double)tid / TABLE + (double)a.q);
  if (tid == ST - 1) {
    sm.n_cand = sm.n_all = 0;
    sm.told[0] = sm.told[1] = 0;
    sm.first = LAST;
    sm.off_min = log2((double)min_p) / r.scale;  // w >= min_p where x >= top + this
    sm.off_low = (a.q + 2.0) / r.scale;          // what is further below rounds to nothing
  }
  for (int i = tid; i < 2 * BINS; i += ST) sm.hist[0][i] = 0;
  asm volatile("cp.async.wait_group 0;" ::: "memory");
  __syncthreads();

  // ---- 1: the largest
  float best = -CUDART_INF_F;  // of this thread's
  {
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
  // (and where `low`, the float below what has a weight, is so far below it that its
  // steps leave the exponents there are: 2^-100 rounds to 0, 2^-900 is still a number)
  r.exact = inf || temp < 0x1p-80f || !(fabs((double)r.top * r.step) < 0x1p50) || !(r.low > -MAXF) || !(((double)r.top - (double)r.low) * r.scale < 900.0);
  if (r.exact) r.step = TABLE, r.none = -CUDART_INF_F;
  else r.zero -= rint((double)r.top * r.step);

  // ---- 2, 3: the cut of top-k, then of top-p
  bool do_k = RULES && top_k > 0 && top_k < a.n, do_p = RULES && top_p < 1.0f;
  // bins of 1/32 nat for top-k: to the nearest, by an addition in which the
  // sum's last bits are the number (what the constant loses shifts all alike).
  // The largest is in bin 0: below 4e6 a product is rounded by 1/8 at the most, so
  // that its floor is no more than 1/8 above the product itself, and bin 0 ends at 1/2.
  const float per_unit = fmaxf(fminf(32.0f / temp, 1e30f), 1e-38f);
  const float bias = fminf(fmaxf(floorf(r.top * per_unit), -4e6f), 4e6f);
  const bool near = fabsf(r.top * per_unit) < 4e6f;
  auto bin_k = [&](float x) {
    const float d = near ? fmaf(x, -per_unit, bias) : x == r.top ? 0.0f : (r.top - x) * per_unit;
    return (int)(__float_as_uint(fminf(fmaxf(d, 0.0f), (float)(BINS - 1)) + 8388608.0f) & 2047u);  // (NaN, of infinities: 0)
  };
  // for top-p by the f32 weight's exponent and five bits: bin 0 is 1; the last
  // one's, below 2^-31, are not counted
  // y = (x - top) scale, with both times `pre`: 1 but where differences may overflow
  // (temperatures past 2^60) or count as subnormals (below 4e-39, of logits below
  // 2^-40; larger ones are 2^-64 apart, which any such slope makes nothing of).  So
  // the slope is finite, and the largest has y = 0 (of infinities NaN, counted as 0).
  const float pre = r.scale < 0x1p-60 ? 0.5f : r.scale > (double)MAXF && fabsf(r.top) < 0x1p-40f ? 0x1p100f : 1.0f;
  const float less = -r.top * pre, slope = inf ? 1.0f : (float)fmin(r.scale / (double)pre, (double)MAXF);
  auto weight_p = [&](float x) {
    const float y = fminf(fmaf(x, pre, less) * slope, 0.0f);
    float w;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(w) : "f"(y));
    return __float_as_uint(w);
  };
  // (unsigned: what would be before bin 0 goes to the last one, so that no bin is out of range)
  auto bin_p = [&](uint32_t w) { return (int)min((127u << 5) - (w >> 18), (uint32_t)(BINS - 1)); };
  float before_x = CUDART_NAN_F;  // logits from here on are before those in question
  u64 sum = 0;                    // their weights and number
  uint32_t n = 0;
  bool maxima = do_k && top_k <= min(ST * a.cluster / 2, 352);  // of the threads' first (which 431 of all pass, on average, at the most)
  for (bool again = false; do_k || do_p; again = true) {
    const bool weigh = !do_k;  // top-p of all that is kept
    if (again) {
      r.sync();  // (the histogram has been read)
      for (int i = tid; i < 2 * BINS; i += ST) sm.hist[0][i] = 0;
      if (tid == 0) sm.n_cand = sm.n_all = 0, sm.told[0] = sm.told[1] = 0;
      __syncthreads();
    }
    uint32_t *hist = sm.hist[lane & 1];
    if (weigh) {
      r.each4([&](const float *x, int i) {
        bool on[4];
        r.kept4(x, i, on);
#pragma unroll
        for (int e = 0; e < 4; e++) {
          const uint32_t w = weight_p(x[e]);
          const int b = bin_p(w);
          if (on[e] && b < BINS - 1) atomicAdd(hist + b, ((w & 0x7fffffu) | 0x800000u) >> a.drop);
        }
      });
    } else if (maxima) {
      if (best >= r.cx) atomicAdd(hist + bin_k(best), 1u);
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
    sm.hist[0][tid + ST] += sm.hist[1][tid + ST];
    if (tid == 0) sm.lo = sm.hi = BINS - 1;
    r.sync();
    // bins 2 tid and 2 tid + 1 of the whole row, and the sums down to them: tokens
    // (for top-p, what they are at the most), weights
    uint32_t c[2] = {0, 0};
    float m[2] = {0.0f, 0.0f};
    {
      u64 v[8];
#pragma unroll
      for (int k = 0; k < 8; k++) v[k] = k < a.cluster ? peer64(&sm.hist[0][2 * tid], k) : 0;
#pragma unroll
      for (int k = 0; k < 8; k++)
#pragma unroll
        for (int j = 0; j < 2; j++) {
          const uint32_t x = (uint32_t)(v[k] >> (32 * j));
          m[j] += (float)x;
          c[j] += weigh ? x >> (23 - a.drop) : x;
        }
#pragma unroll
      for (int j = 0; j < 2; j++) m[j] *= exp2f((float)(-((2 * tid + j + 31) >> 5)));
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
    // (sums of weights need not ascend by the last bit: the first bin that passes)
    const uint32_t k = (uint32_t)max(top_k, 1);
    uint32_t l = BINS - 1, h = BINS - 1;
#pragma unroll
    for (int j = 1; j >= 0; j--) {
      const uint32_t cj = j ? cs : cs - c[1];
      const float mj = j ? ms : ms - m[1];
      if (do_k ? cj >= k : mj >= mass * top_p * (1.0f - a.margin)) l = 2 * tid + j;
      if (do_k ? cj >= k : mj >= mass * top_p * (1.0f + a.margin)) h = 2 * tid + j;
    }
    l = __reduce_min_sync(0xffffffffu, l);
    h = __reduce_min_sync(0xffffffffu, h);
    if (lane == 0 && l < BINS - 1) atomicMin(&sm.lo, l);
    if (lane == 0 && h < BINS - 1) atomicMin(&sm.hi, h);
    __syncthreads();
    const int hi = (int)sm.hi;
    int lo = (int)sm.lo;
    if (tid == hi / 2) sm.at = hi & 1 ? cs : cs - c[1];
    if (tid == lo / 2) sm.above = cs - c[1] - (lo & 1 ? 0 : c[0]);
    __syncthreads();
    if (do_k && !maxima && k >= total && total > CAP) {  // top-k keeps them all
      do_k = false;
      continue;
    }
    uint32_t above = sm.above;  // tokens before bin lo (top-k of all)
    const bool whole = maxima || (sm.at <= CAP && (do_k || hi < BINS - 1));  // all down to there, if they are few
    if (whole) lo = 0, above = 0;
    // The least floats of bins below lo (that are before those in question) and
    // of bins up to hi, a warp each: 33 floats around where the bin should end,
    // or, if it does not there, 33 that divide all, and so on.
    if (warp < 2) {
      const int b = warp == 0 ? lo - 1 : hi;
      auto in = [&](uint32_t key) {
        const float x = of_key(key);
        return (do_k ? bin_k(x) : bin_p(weight_p(x))) <= b;
      };
      const uint32_t least = key_of(-CUDART_INF_F);
      uint32_t from = least, to = key_of(r.top);  // (of which one is not looked at, the other is in bin 0)
      if (b < 0 || b == BINS - 1) {
        from = to = b < 0 ? 0 : key_of(-MAXF);
      } else {
        const double g = do_k ? ((double)bias - b - 0.5) / (double)per_unit
                              : (double)r.top + (double)log2f(__uint_as_float((uint32_t)((127 << 5) - b) << 18)) / r.scale;
        const uint32_t at = min(max(key_of((float)g), least + 17), to - min(to - least - 17, 16u));
        const bool here = lane == 0 ? !in(at - 16) : lane == 1 ? in(at + 16) : true;
        if (to - least > 64 && __all_sync(0xffffffffu, here)) from = at - 16, to = at + 16;
      }
      while (to - from > 1) {
        const uint32_t step = (to - from + 31) / 32, at = from + min((uint32_t)(lane + 1) * step, to - from);
        const uint32_t lanes = __ballot_sync(0xffffffffu, in(at));  // (`to` is among them: the largest is in bin 0)
        if (!lanes) break;
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

    // ---- 3
    const uint32_t to = map_rank(shaddr(&sm.cand[0]), 0), counter = map_rank(shaddr(&sm.n_cand), 0);
    uint32_t taken = 0;
    auto take = [&](float x, int i) {
      uint32_t at;
      asm volatile("atom.relaxed.cluster.shared::cluster.add.u32 %0, [%1], 1;" : "=r"(at) : "r"(counter) : "memory");
      if (at < CAP) asm volatile("st.shared::cluster.u64 [%0], %1;" ::"r"(to + at * 8), "l"(order_of(x, i)) : "memory");
      taken++;
    };
    // so that every CTA has the number of all that were taken
    auto tell_taken = [&]() {
      taken = __reduce_add_sync(0xffffffffu, taken);
      if (taken && lane < a.cluster) asm volatile("red.relaxed.cluster.shared::cluster.add.u32 [%0], %1;" ::"r"(map_rank(shaddr(&sm.n_all), lane)), "r"(taken) : "memory");
    };
    u64 weight = 0;
    sum = 0;
    n = 0;
    if (weigh) {
      const bool plain = r.ci == LAST && r.cx <= r.none;  // nothing is cut off that has a weight
      auto pass = [&](auto ex, auto pl) {
        constexpr bool EX = decltype(ex)::value, PL = decltype(pl)::value;
        uint32_t made = 0, made_before = 0;
        r.each4([&](const float *x, int i) {
          bool on[4];
          float y[4];
          if (!PL) r.kept4(x, i, on);
#pragma unroll
          for (int e = 0; e < 4; e++) {
            y[e] = fmaxf(x[e], r.none);
            if (!PL && !on[e]) y[e] = r.none;
            const u64 w = r.raw(r.template weight_as<EX>(y[e]));
            weight += w;
            if (y[e] >= before_x) sum += w, made_before++;
          }
          made += 4;
          if (fmaxf(fmaxf(y[0], y[1]), fmaxf(y[2], y[3])) >= last_x) {
#pragma unroll
            for (int e = 0; e < 4; e++)
              if (y[e] >= last_x && !(y[e] >= before_x) && (PL || on[e])) take(x[e], i + e);
          }
        });
        weight -= made * r.ONE;
        sum -= made_before * r.ONE;
        n = made_before;
      };
      if (r.exact) pass(std::true_type{}, std::false_type{});
      else if (plain) pass(std::false_type{}, std::true_type{});
      else pass(std::false_type{}, std::false_type{});
      tell_taken();
      const u64 w0 = r.sum_warp(weight), w1 = r.sum_warp(sum);
      if (lane == 0) sm.warp[warp] = w0, sm.warpb[warp] = w1;
      __syncthreads();
      if (warp < 2) {
        const u64 v = r.sum_warp(lane < SW ? (warp ? sm.warpb : sm.warp)[lane] : 0);
        if (lane < a.cluster) asm volatile("red.relaxed.cluster.shared::cluster.add.u64 [%0], %1;" ::"r"(map_rank(shaddr(&sm.told[warp]), lane)), "l"(v) : "memory");
      }
    } else {
      r.each4([&](const float *x, int i) {
        if (!(x[0] >= last_x || x[1] >= last_x || x[2] >= last_x || x[3] >= last_x)) return;
#pragma unroll
        for (int e = 0; e < 4; e++)
          if (x[e] >= last_x && !(x[e] >= before_x) && r.kept(x[e], i + e)) take(x[e], i + e);
      });
      tell_taken();
    }
    r.sync();
    uint32_t inside = sm.n_all;
    if (maxima && inside > CAP) {  // (equal logits, or thousands near the threads' k-th)
      maxima = false;
      continue;
    }
    if (whole && inside <= CAP && rank > 0) return;  // (the first CTA has all that it needs)
    weight = sm.told[0];
    u64 base_w = sm.told[1];
    const double target = (double)top_p * (double)weight;
    const bool many = inside > CAP;
    if (many) {
      // The order's range is narrowed to one of 512 parts of it at a time, by their
      // numbers of tokens and exact weights (seven times at the most).
      u64 o_lo = order_of(last_x, LAST), o_hi = order_of(before_x == before_x ? before_x : r.top, 0);
      uint32_t *part_n = sm.hist[0];
      u64 *part_w = reinterpret_cast<u64 *>(sm.hist[1]);
      static_assert(sizeof(sm.hist[1]) >= ST * sizeof(u64), "room");
      auto asked = [&](float x, int i) {
        if (!(x >= last_x) || x >= before_x || !r.kept(x, i)) return false;
        const u64 o = order_of(x, i);
        return o >= o_lo && o <= o_hi;
      };
      for (int turn = 0; inside > CAP && turn < 8; turn++) {
        const int shift = max(0, 64 - 9 - __clzll((long long)(o_hi - o_lo)));
        part_n[tid] = 0;
        part_w[tid] = 0;
        __syncthreads();
        r.each_warp([&](const float *x, int i) {
#pragma unroll
          for (int e = 0; e < 4; e++) {
            const bool on = asked(x[e], i + e);
            const uint32_t lanes = __ballot_sync(0xffffffffu, on);
            if (!lanes) continue;
            const int part = (int)((o_hi - order_of(x[e], i + e)) >> shift);
            const u64 w = on && weigh ? r.fixed(x[e]) : 0;
            // (equal logits by thousands are in one part: one addition a warp)
            const int first = __shfl_sync(0xffffffffu, part, __ffs(lanes) - 1);
            if (__all_sync(0xffffffffu, !on || part == first)) {
              const u64 all_w = r.sum_warp(w);
              if (lane == 0) {
                atomicAdd(part_n + first, (uint32_t)__popc(lanes));
                if (weigh) atomicAdd(part_w + first, all_w);
              }
            } else if (on) {
              atomicAdd(part_n + part, 1u);
              if (weigh) atomicAdd(part_w + part, w);
            }
          }
        });
        r.sync();
        uint32_t c = 0;
        u64 w = 0;
        for (int j = 0; j < a.cluster; j++) c += peer32(part_n + tid, j), w += peer64(part_w + tid, j);
        uint32_t cs = c;
#pragma unroll
        for (int i = 1; i < 32; i *= 2) {
          const uint32_t y = __shfl_up_sync(0xffffffffu, cs, i);
          if (lane >= i) cs += y;
        }
        if (lane == 31) sm.warp2[warp] = cs;
        if (tid == 0) sm.at = ~0u;
        const u64 wb = base_w + r.scan(w);  // (its barriers order warp2 and at, too)
        uint32_t cb = above + cs - c, all_c = above;
        for (int i = 0; i < SW; i++) {
          if (i < warp) cb += sm.warp2[i];
          all_c += sm.warp2[i];
        }
        // the part with which the goal is reached; if none does, the last one
        if (c && (do_k ? cb < k && cb + c >= k : (double)wb < target && (double)(wb + w) >= target)) sm.at = (uint32_t)tid, sm.above = cb, sm.inside = c, sm.base_w = wb;
        __syncthreads();
        const bool none = sm.at == ~0u;
        __syncthreads();
        if (none && c && cb + c == all_c) sm.at = (uint32_t)tid, sm.above = cb, sm.inside = c, sm.base_w = wb;
        __syncthreads();
        const u64 to = o_hi - ((u64)sm.at << shift), span = (1ull << shift) - 1;
        o_lo = to - o_lo > span ? to - span : o_lo;
        o_hi = to;
        above = sm.above;
        inside = sm.inside;
        base_w = sm.base_w;
        r.sync();  // (the parts have been read)
      }
      if (tid == 0) sm.n_cand = 0;
      r.sync();
      r.each([&](float x, int i) {
        if (asked(x, i)) take(x, i);
      });
      r.sync();
    }
    const bool last = whole && !many;  // the first CTA goes on to the token
    if (rank == 0) {
      const int nc = min((int)sm.n_cand, CAP);
      if (nc <= FEW) {
        if (warp == 0) {
          auto few = [&](auto j) {
            constexpr int J = decltype(j)::value;
            u64 v[J], w[J], s[J];
#pragma unroll
            for (int i = 0; i < J; i++) v[i] = 32 * i + lane < nc ? sm.cand[32 * i + lane] : 0;
            sort_warp(v, lane);
            int cut = do_k ? min(nc, (int)(k - above)) : nc;  // how many are kept
            if (!do_k || last) {
#pragma unroll
              for (int i = 0; i < J; i++) s[i] = w[i] = 32 * i + lane < cut ? r.fixed(of_key((uint32_t)(v[i] >> 32))) : 0;
              scan_warp(s, lane);
              if (do_p) {  // up to the first with which they have top_p of the weight
                const double goal = do_k ? (double)top_p * (double)__shfl_sync(0xffffffffu, s[J - 1], 31) : target;
                int first = cut - 1;
#pragma unroll
                for (int i = J - 1; i >= 0; i--) {
                  const uint32_t lanes = __ballot_sync(0xffffffffu, 32 * i + lane < cut && (double)(base_w + s[i]) >= goal);
                  if (lanes) first = 32 * i + __ffs(lanes) - 1;
                }
                cut = first + 1;
              }
            }
            if (!last) {
#pragma unroll
              for (int i = 0; i < J; i++)
                if (32 * i + lane == cut - 1) sm.cut_x = of_key((uint32_t)(v[i] >> 32)), sm.cut_i = (int)~(uint32_t)v[i];
              return;
            }
            // the kept ones by index (the largest first: from the least ~index on), and the one where u falls
            u64 *few_w = reinterpret_cast<u64 *>(sm.hist[1]), all_w = 0;
#pragma unroll
            for (int i = 0; i < J; i++) {
              const int at = 32 * i + lane;
              if (at < cut) all_w += w[i];
              few_w[at] = w[i];
              v[i] = at < cut ? (u64)(uint32_t)v[i] << 10 | (uint32_t)at : 0;
            }
            __syncwarp();
            all_w = r.sum_warp(all_w);
            sort_warp(v, lane);
#pragma unroll
            for (int i = 0; i < J; i++) s[i] = w[i] = v[i] ? few_w[v[i] & 1023] : 0;
            scan_warp(s, lane);
            const u64 pass = pass_of(u, all_w);
#pragma unroll
            for (int i = 0; i < J; i++)
              if (w[i] && pass < s[i] && pass >= s[i] - w[i]) {
                a.p.tok[row] = (int)~(uint32_t)(v[i] >> 10);
                if (a.p.prob) a.p.prob[row] = (float)((double)w[i] / (double)all_w);
                if (a.p.kept) a.p.kept[row] = cut;
              }
          };
          if (nc <= 32) few(std::integral_constant<int, 1>{});
          else if (nc <= 64) few(std::integral_constant<int, 2>{});
          else few(std::integral_constant<int, 4>{});
        }
      } else {
        // the same with a thread for each
        u64 v = r.sorted(tid < nc ? sm.cand[tid] : 0, nc);
        int cut = do_k ? min(nc, (int)(k - above)) : nc;
        u64 w = 0, all_w = 0;
        if (!do_k || last) {
          w = tid < cut ? r.fixed(of_key((uint32_t)(v >> 32))) : 0;
          const u64 b = r.scan(w);
          if (tid == ST - 1) sm.x[4] = b + w;
          if (tid == 0) sm.at = (uint32_t)cut - 1;
          __syncthreads();
          all_w = sm.x[4];
          __syncthreads();
          if (do_p) {
            const double goal = do_k ? (double)top_p * (double)all_w : target;
            if (tid < cut && (double)(base_w + b + w) >= goal && (tid == 0 || (double)(base_w + b) < goal)) sm.at = (uint32_t)tid, sm.x[4] = b + w;
            __syncthreads();
            cut = (int)sm.at + 1;
            all_w = sm.x[4];
          }
        }
        if (!last) {
          if (tid == cut - 1) sm.cut_x = of_key((uint32_t)(v >> 32)), sm.cut_i = (int)~(uint32_t)v;
        } else {
          u64 *few_w = reinterpret_cast<u64 *>(sm.hist[1]);
          few_w[tid] = w;
          v = r.sorted(tid < cut ? (u64)(uint32_t)v << 10 | (uint32_t)tid : 0, cut);
          w = v ? few_w[v & 1023] : 0;
          const u64 b = r.scan(w), pass = pass_of(u, all_w);
          if (w && pass >= b && pass < b + w) {
            a.p.tok[row] = (int)~(uint32_t)(v >> 10);
            if (a.p.prob) a.p.prob[row] = (float)((double)w / (double)all_w);
            if (a.p.kept) a.p.kept[row] = cut;
          }
        }
      }
      if (last) return;
    }
    r.sync();
    r.cx = __uint_as_float(peer32(&sm.cut_x, 0));
    r.ci = (int)peer32(&sm.cut_i, 0);
    if (do_k) do_k = maxima = false;
    else do_p = false;
  }

  // ---- 4: the kept weights by index (of what came before top-p's tokens in question they are there)
  if (!(top_p < 1.0f)) sum = 0, n = 0, before_x = CUDART_NAN_F;
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
        // (most are neither: that first)
        bool on[4], any = false;
#pragma unroll
        for (int e = 0; e < 4; e++) any |= x[e] >= r.cx && !(RULES && x[e] >= before_x);
        if (!any) return;
        r.kept4(x, i, on);
#pragma unroll
        for (int e = 0; e < 4; e++) {
          if (RULES) on[e] = on[e] && !(x[e] >= before_x);
          n += on[e] ? 1 : 0;
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
  const u64 pass = pass_of(u, all_w);
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
  // CTAs a row: by what they hold, two an SM, one where rows are longer; more
  // where the rows leave SMs without any.  (250 f32 rows of 128256, each with its
  // own rules: 5 CTAs 149 us, 6 156, 4 (one an SM) 189, and read again from L2 for
  // every pass, 2 195 and one 288, which waits for the longest row; 64 bf16 rows of
  // 73448: 4 CTAs 41, 2 55, 6 60.)
  const long long vecs = ((long long)n + 2 * v - 2) / v, most = (113 * 1024 - (int)sizeof(Smem)) / 16, wide = 208 * 1024 / 16;
  long long c = std::min(8LL, (vecs + most - 1) / most);
  while (c < 8 && rows * c * 2 <= 296 && vecs >= 512 * c) c *= 2;
  c = std::min(c, 8LL);
  const long long seg = (vecs + c - 1) / c;
  const bool big = seg > wide;
  a.cluster = (int)c;
  a.seg = (int)(seg * v);
  // 24 bits of a weight, of which 16 are kept: 65536 of a bin and CTA fit 32 bits
  a.drop = 8;
  for (long long x = 65536; x < a.seg; x *= 2) a.drop++;
  a.margin = MARGIN + (float)(1 << a.drop) * 0x1p-23f + (float)n * 0x1p-31f;  // (the last bin's weights are left out)
  const int smem = (int)sizeof(Smem) + (big ? 0 : (int)(seg * 16));
  const dim3 grid((unsigned)(rows * c)), block(ST);
  const bool rules = p.top_k || p.top_p || p.min_p;
#define GO(E) launch_cluster(rules ? big ? k_sample<E, true, true> : k_sample<E, false, true> : big ? k_sample<E, true, false> : k_sample<E, false, false>, (int)c, grid, block, smem, st, a)
  return type == T_F32 ? GO(float) : type == T_F16 ? GO(__half) : GO(__nv_bfloat16);
#undef GO
}

}  // namespace pk
