// What the attention kernels of 128-row tcgen05 tiles share: operand descriptors of swizzled
// tiles, exponentials and row stores.
#pragma once

#include "sm100_common.cuh"

namespace tfb {

constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLn2 = 0.6931471805599453f;
constexpr uint32_t kPanel = 128u * 128u;  // one 64-column panel of 128 rows (bytes)

// K-major operand tile with K = 128 elements (two 64-element panels): k-step kk of 16.
__device__ __forceinline__ uint64_t desc_kmajor(uint32_t base, int kk) {
  return umma_desc_sw128(base + (uint32_t)(kk >> 2) * kPanel + (uint32_t)(kk & 3) * 32u, 16, 1024);
}
// MN-major operand tile (MN in 64-element panels, K along the 128 rows): k-step kk of 16.
__device__ __forceinline__ uint64_t desc_mnmajor(uint32_t base, int kk) {
  return umma_desc_sw128(base + (uint32_t)kk * 2048u, kPanel, 1024);
}

__device__ __forceinline__ void store_row_bf16_global(__nv_bfloat16* dst, const float* v, int n) {
  for (int c = 0; c < n / 8; ++c) {
    uint4 u;
    u.x = pack_bf16x2(v[8 * c + 0], v[8 * c + 1]);
    u.y = pack_bf16x2(v[8 * c + 2], v[8 * c + 3]);
    u.z = pack_bf16x2(v[8 * c + 4], v[8 * c + 5]);
    u.w = pack_bf16x2(v[8 * c + 6], v[8 * c + 7]);
    reinterpret_cast<uint4*>(dst)[c] = u;
  }
}

__device__ __forceinline__ float ex2_approx(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

__device__ __forceinline__ float max3f(float a, float b, float c) {
  float d;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
  return d;
}

// max that keeps a NaN
__device__ __forceinline__ float max3_nan(float a, float b, float c) {
  float d;
  asm("max.NaN.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
  return d;
}
__device__ __forceinline__ float max_nan(float a, float b) {
  float d;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(d) : "f"(a), "f"(b));
  return d;
}

// 2^v on the FMA pipe for v <= 8 (0 below -126): v = n + f with n the nearest integer
// (added and subtracted 1.5 * 2^23, whose low mantissa bits then hold n) and f in
// [-1/2, 1/2]; 2^f from a degree-3 polynomial fitted here for relative error on that
// interval (max relative error 7.5e-5, far below the bf16 rounding of P); 2^n added
// into the exponent field as n << 23, which is the magic sum's bits shifted by 23.
// Clamping v at -126 keeps that exponent field from underflowing.
__device__ __forceinline__ float2 exp2_poly2(float2 v) {
  const float2 vc = make_float2(fmaxf(v.x, -126.f), fmaxf(v.y, -126.f));
  const float2 t = __fadd2_rn(vc, make_float2(12582912.f, 12582912.f));
  const float2 n = __fadd2_rn(t, make_float2(-12582912.f, -12582912.f));
  const float2 f = __fadd2_rn(vc, make_float2(-n.x, -n.y));
  float2 p = __ffma2_rn(make_float2(0.055170949548482895f, 0.055170949548482895f), f,
                        make_float2(0.2426096349954605f, 0.2426096349954605f));
  p = __ffma2_rn(p, f, make_float2(0.6932609677314758f, 0.6932609677314758f));
  p = __ffma2_rn(p, f, make_float2(0.9999281764030457f, 0.9999281764030457f));
  const float rx = __int_as_float(__float_as_int(p.x) + (__float_as_int(t.x) << 23));
  const float ry = __int_as_float(__float_as_int(p.y) + (__float_as_int(t.y) << 23));
  return make_float2(v.x < -126.f ? 0.f : rx, v.y < -126.f ? 0.f : ry);
}

// 32 lanes x 16 consecutive 32-bit TMEM columns.
__device__ __forceinline__ void tmem_ld_32x32b_x16(uint32_t taddr, uint32_t (&r)[16]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]),
        "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
      : "r"(taddr));
}
__device__ __forceinline__ void tmem_st_32x32b_x16(uint32_t taddr, const uint32_t (&r)[16]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16};" ::"r"(taddr),
      "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]),
      "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15])
      : "memory");
}

}  // namespace tfb
