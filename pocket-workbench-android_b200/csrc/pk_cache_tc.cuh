// pk_cache_tc.cuh -- what the two tcgen05 kernels of the attention over the
// quantised cache share (pk_cache_attn_tc.cu, pk_cache_prefix.cu).
#pragma once
#include <type_traits>

#include "pk_cache_attn.cuh"
#include "pk_tcgen05.cuh"

namespace pk {
namespace {

constexpr unsigned long long WAIT_NS = 2000000000ull;

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

// The same on pairs that stay in a 64-bit register: what is used again and again
// is packed once.
__device__ __forceinline__ uint64_t pair_of(float a, float b) {
  uint64_t d;
  asm("mov.b64 %0, {%1, %2};" : "=l"(d) : "f"(a), "f"(b));
  return d;
}
__device__ __forceinline__ float2 unpair(uint64_t a) {
  float2 d;
  asm("mov.b64 {%0, %1}, %2;" : "=f"(d.x), "=f"(d.y) : "l"(a));
  return d;
}
__device__ __forceinline__ uint64_t mul2(uint64_t a, uint64_t b) {
  uint64_t d;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
  return d;
}
__device__ __forceinline__ uint64_t add2(uint64_t a, uint64_t b) {
  uint64_t d;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
  return d;
}
__device__ __forceinline__ uint64_t fma2(uint64_t a, uint64_t b, uint64_t c) {
  uint64_t d;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(d) : "l"(a), "l"(b), "l"(c));
  return d;
}

// The order of a word's eight dimensions in an operand: as they lie for Q8, as
// the nibble pairs (i, i + 4) come out for Q4.
template <int TYPE>
__host__ __device__ constexpr int dim8(int i) {
  return TYPE == PK_KV_Q8 ? i : (i / 2) + 4 * (i % 2);
}

// A query row into the operand by two threads, half of it each (half precision):
// f16 as it is, bf16 scaled to |q'| < 2 and rounded to f16 (exact down to 2^-24
// of the row's largest); returns its scale (the D^K that the row meets have
// log2(e) * scale in them).
template <int TYPE, int DH, class E>
__device__ __forceinline__ float put_q_half(const AttnKArgs &a, const Unit &u, int row, int part, uint32_t dst, int stride) {
  constexpr bool F16 = std::is_same_v<E, __half>;
  constexpr int N = DH / 16;  // vectors of 8
  const bool on = row < u.rows;
  const int i = row / a.group, h = u.h * a.group + row - i * a.group;
  const E *p = reinterpret_cast<const E *>(a.q.q) + (on ? (long long)(u.sv.first + i) * a.q.q_tok_stride + (long long)h * a.q.q_head_stride : 0) + part * (DH / 2);
  uint4 raw[N];
  const E *x = reinterpret_cast<const E *>(raw);
  if (on && a.vec_q) {
#pragma unroll
    for (int c = 0; c < N; c++) raw[c] = __ldg(reinterpret_cast<const uint4 *>(p) + c);
  } else {
    E *y = reinterpret_cast<E *>(raw);
#pragma unroll
    for (int j = 0; j < 8 * N; j++) y[j] = on ? p[j] : from_f<E>(0.0f);
  }
  float m = 0.0f;
  if (!F16) {
#pragma unroll
    for (int j = 0; j < 8 * N; j++) m = fmaxf(m, fabsf(to_f(x[j])));
    m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, 1));
  }
  int e = (int)(__float_as_uint(m) >> 23) - 127;
  e = m > 0.0f ? min(max(e, -100), 126) : 0;
  const float up = __int_as_float((e + 127) << 23), down = __int_as_float((127 - e) << 23);
#pragma unroll
  for (int c = 0; c < N; c++) {
    uint32_t w[4];
#pragma unroll
    for (int j = 0; j < 4; j++)
      w[j] = pack2(inf_nan(to_f(x[8 * c + dim8<TYPE>(2 * j)])) * down, inf_nan(to_f(x[8 * c + dim8<TYPE>(2 * j + 1)])) * down);
    sts128(dst + (part * N + c) * stride, w[0], w[1], w[2], w[3]);
  }
  return up;
}

}  // namespace
}  // namespace pk
