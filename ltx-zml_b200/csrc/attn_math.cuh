// Arithmetic shared by the tcgen05 attention kernels (attn_tc.cu,
// kv4_attn_tc.cu): exp2 on the MUFU and FMA pipes, two-wide f32 operations,
// and MMA issue from descriptor low words.
#pragma once

#include "common.cuh"

namespace ltxb {

__device__ __forceinline__ float ex2_mufu(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// 2^x on the FMA pipe: x = n + f with n = rint(x) (via the 1.5 * 2^23
// rounding constant), f in [-1/2, 1/2]; 2^f by a degree-3 polynomial fitted by
// least squares on Chebyshev nodes of [-1/2, 1/2] (max relative error
// 7.8e-5); 2^n is added to the exponent field. x is clamped to >= -120, which
// keeps the exponent arithmetic in range (2^-120 is negligible next to a
// row sum >= 1).
__device__ __forceinline__ float ex2_poly(float x) {
  x = fmaxf(x, -120.0f);
  const float magic = 12582912.0f;  // 1.5 * 2^23
  const float t = x + magic;
  const float n = t - magic;
  const float f = x - n;
  float p = fmaf(0.05508868396282196f, f, 0.24260404706001282f);
  p = fmaf(p, f, 0.6932762265205383f);
  p = fmaf(p, f, 0.9999289512634277f);
  return __int_as_float(__float_as_int(p) + (__float_as_int(t) << 23));
}

// Two-wide f32 SIMD (sm_100 `*.f32x2`) on register pairs.
__device__ __forceinline__ uint64_t pk2(float a, float b) {
  uint64_t r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ void up2(uint64_t v, float& a, float& b) {
  asm("mov.b64 {%0, %1}, %2;" : "=f"(a), "=f"(b) : "l"(v));
}
__device__ __forceinline__ uint64_t fma2(uint64_t a, uint64_t b, uint64_t c) {
  uint64_t r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
  return r;
}
__device__ __forceinline__ uint64_t add2(uint64_t a, uint64_t b) {
  uint64_t r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
__device__ __forceinline__ float max3(float a, float b, float c) {
  float r;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
  return r;
}

// MMA issue with the shared-memory descriptors passed as their low words: the
// high word of every 128-byte-swizzle descriptor here is the same constant
// (SBO 1024 B, descriptor version 1, layout SWIZZLE_128B), and the low word
// (start address >> 4, LBO) is stepped by plain 32-bit adds.
constexpr uint32_t kDescHi = (1024u >> 4) | (1u << 14) | (2u << 29);
__device__ __forceinline__ uint32_t desc_lo(uint32_t saddr, uint32_t lbo_field) {
  return ((saddr >> 4) & 0x3FFFu) | (lbo_field << 16);
}
__device__ __forceinline__ void mma_ss_lo(uint32_t d, uint32_t alo, uint32_t blo, uint32_t idesc, uint32_t acc) {
  asm volatile(
      "{\n\t.reg .b64 da, db;\n\t.reg .pred p;\n\t"
      "mov.b64 da, {%1, %5};\n\tmov.b64 db, {%2, %5};\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], da, db, %3, p;\n\t}" ::"r"(d),
      "r"(alo), "r"(blo), "r"(idesc), "r"(acc), "r"(kDescHi)
      : "memory");
}
__device__ __forceinline__ void mma_ts_lo(uint32_t d, uint32_t a_tmem, uint32_t blo, uint32_t idesc, uint32_t acc) {
  asm volatile(
      "{\n\t.reg .b64 db;\n\t.reg .pred p;\n\t"
      "mov.b64 db, {%2, %5};\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], db, %3, p;\n\t}" ::"r"(d),
      "r"(a_tmem), "r"(blo), "r"(idesc), "r"(acc), "r"(kDescHi)
      : "memory");
}

// ex2_poly for a pair, the range reduction and polynomial in f32x2.
__device__ __forceinline__ void ex2_poly2(float x0, float x1, float& p0, float& p1) {
  x0 = fmaxf(x0, -120.0f);
  x1 = fmaxf(x1, -120.0f);
  const uint64_t x2 = pk2(x0, x1);
  const uint64_t t2 = add2(x2, pk2(12582912.0f, 12582912.0f));
  const uint64_t n2 = add2(t2, pk2(-12582912.0f, -12582912.0f));
  const uint64_t f2 = fma2(n2, pk2(-1.0f, -1.0f), x2);
  uint64_t q2 = fma2(pk2(0.05508868396282196f, 0.05508868396282196f), f2,
                     pk2(0.24260404706001282f, 0.24260404706001282f));
  q2 = fma2(q2, f2, pk2(0.6932762265205383f, 0.6932762265205383f));
  q2 = fma2(q2, f2, pk2(0.9999289512634277f, 0.9999289512634277f));
  float t0, t1;
  up2(q2, p0, p1);
  up2(t2, t0, t1);
  p0 = __int_as_float(__float_as_int(p0) + (__float_as_int(t0) << 23));
  p1 = __int_as_float(__float_as_int(p1) + (__float_as_int(t1) << 23));
}

}  // namespace ltxb
