// Device helpers of the tcgen05 attention kernels: tensor-memory stores, the
// product with A in tensor memory, and the exponentials of the softmax.
#pragma once

#include "common.cuh"

namespace dcpp {

__device__ __forceinline__ void tmem_st32(uint32_t taddr, const uint32_t* r) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x32.b32 [%0],"
      " {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,"
      "%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31,%32};" ::"r"(taddr),
      "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]),
      "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]), "r"(r[16]),
      "r"(r[17]), "r"(r[18]), "r"(r[19]), "r"(r[20]), "r"(r[21]), "r"(r[22]), "r"(r[23]), "r"(r[24]),
      "r"(r[25]), "r"(r[26]), "r"(r[27]), "r"(r[28]), "r"(r[29]), "r"(r[30]), "r"(r[31])
      : "memory");
}
__device__ __forceinline__ void tmem_st16(uint32_t taddr, const uint32_t* r) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0],"
      " {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16};" ::"r"(taddr),
      "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]),
      "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15])
      : "memory");
}
__device__ __forceinline__ void tmem_ld16(uint32_t taddr, uint32_t (&r)[16]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x16.b32"
      " {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]),
        "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
      : "r"(taddr));
}
__device__ __forceinline__ void tmem_st_wait() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

// O (+)= A[tmem] * B[smem desc]^T, A (M x K bf16) read from TMEM.
__device__ __forceinline__ void umma_bf16_ts(uint32_t tmem_d, uint32_t tmem_a, uint64_t bdesc, uint32_t idesc,
                                             uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}" ::"r"(tmem_d),
      "r"(tmem_a), "l"(bdesc), "r"(idesc), "r"(accumulate)
      : "memory");
}

__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// Packed f32x2 arithmetic (two lanes of a 64-bit register per instruction).
__device__ __forceinline__ uint64_t f2(float lo, float hi) {
  return (static_cast<uint64_t>(__float_as_uint(hi)) << 32) | __float_as_uint(lo);
}
__device__ __forceinline__ float f2lo(uint64_t v) { return __uint_as_float(static_cast<uint32_t>(v)); }
__device__ __forceinline__ float f2hi(uint64_t v) { return __uint_as_float(static_cast<uint32_t>(v >> 32)); }
__device__ __forceinline__ uint64_t fma2(uint64_t a, uint64_t b, uint64_t c) {
  uint64_t d;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(d) : "l"(a), "l"(b), "l"(c));
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
__device__ __forceinline__ float max3(float a, float b, float c) {
  float d;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
  return d;
}

// 2^x of a pair on the FMA / integer pipes, for a share of the softmax exponentials
// (the MUFU unit alone would limit the softmax: one ex2 per 512 tensor
// FLOPs is exactly its throughput).  Range reduction x = n + f with
// n = round(x) (the 1.5 * 2^23 rounding trick: t holds n in its low bits), f in
// [-1/2, 1/2]; 2^f by a degree-3 polynomial fitted here to minimise the maximum
// relative error on that interval (7.5e-5: 1/52 of a half step of bf16, 1/7 to 1/3 of one of f16).
__device__ __forceinline__ uint64_t ex2_poly2_reduced(uint64_t x, uint64_t& t) {
  const uint64_t magic = f2(12582912.0f, 12582912.0f), neg_magic = f2(-12582912.0f, -12582912.0f);
  t = add2(x, magic);
  const uint64_t n = add2(t, neg_magic);
  const uint64_t f = fma2(n, f2(-1.0f, -1.0f), x);
  uint64_t p = fma2(f2(0.0551716648f, 0.0551716648f), f, f2(0.24261114f, 0.24261114f));
  p = fma2(p, f, f2(0.693260968f, 0.693260968f));
  return fma2(p, f, f2(0.999928057f, 0.999928057f));
}

// 2^n is added to the exponent field.  x is clamped to -126 (masked keys give
// ~2^-126 instead of 0, which vanishes in bf16 sums of O(1) terms).
__device__ __forceinline__ uint64_t ex2_poly2(uint64_t x) {
  x = f2(fmaxf(f2lo(x), -126.0f), fmaxf(f2hi(x), -126.0f));
  uint64_t t;
  const uint64_t p = ex2_poly2_reduced(x, t);
  const uint32_t lo = static_cast<uint32_t>(p) + ((static_cast<uint32_t>(t) - 0x4B400000u) << 23);
  const uint32_t hi = static_cast<uint32_t>(p >> 32) + ((static_cast<uint32_t>(t >> 32) - 0x4B400000u) << 23);
  return (static_cast<uint64_t>(hi) << 32) | lo;
}

// The same with a true 0 for -infinity and everything below -126.5: a masked key's
// value may be as large as the type allows (2^-126 of 3e38 is 3.5).  x is clamped to
// -127, and 2^n is a factor built in the exponent field, which is 0 for n = -127; one
// product more a pair.
__device__ __forceinline__ uint64_t ex2_poly2_zero(uint64_t x) {
  x = f2(fmaxf(f2lo(x), -127.0f), fmaxf(f2hi(x), -127.0f));
  uint64_t t;
  const uint64_t p = ex2_poly2_reduced(x, t);
  const uint32_t lo = (static_cast<uint32_t>(t) << 23) + 0x3F800000u;  // the trick's own bits leave at the top
  const uint32_t hi = (static_cast<uint32_t>(t >> 32) << 23) + 0x3F800000u;
  return mul2(p, (static_cast<uint64_t>(hi) << 32) | lo);
}

}  // namespace dcpp
