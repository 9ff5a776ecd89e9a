// e4m3 codes with a scale: conversions shared by the quantised latent cache, the attention over it and the
// block-scaled products.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_fp8.h>

#include "b200dsa_common.cuh"

namespace b200dsa {

constexpr int kLatentRowBytes = 656;   // 512 codes, 4 fp32 scales, 64 bf16 position dims

// max that keeps a NaN (fmaxf drops it)
__device__ __forceinline__ float max_nan(float a, float b) {
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}

// Smallest power of two that is >= x (x positive): exp2(ceil(log2(x))) on the bit pattern.
__device__ __forceinline__ float pow2_at_least(float x) {
  const uint32_t u = __float_as_uint(x);
  uint32_t e = u >> 23;
  if (e == 0) return 1.17549435e-38f;   // subnormal: the smallest normal power of two
  if (e == 255) return x;               // infinity and NaN stay what they are
  if (u & 0x7fffffu) ++e;
  return __uint_as_float(e << 23);
}

// The scale of a group whose largest value is amax (not below the format's floor) and its reciprocal, for the e4m3 range
// of 448 = 1.75 * 2^8: amax / 448, or the smallest power of two that is not below it, which the bits of amax give (its
// exponent less 8, one more above 1.75) without a division.  An infinite amax gives an infinite scale.
struct GroupScale {
  float scale, rcp;
};
__device__ __forceinline__ GroupScale group_scale_pow2(float amax) {
  const uint32_t u = __float_as_uint(amax);
  const uint32_t e = (u >> 23) - 8u + ((u & 0x7fffffu) > 0x600000u ? 1u : 0u);
  GroupScale g;
  g.scale = u < 0x7f800000u ? __uint_as_float(e << 23) : amax;
  g.rcp = u < 0x7f800000u ? __uint_as_float((254u - e) << 23) : 0.f;
  return g;
}
__device__ __forceinline__ GroupScale group_scale(float amax) {
  GroupScale g;
  g.scale = __fdiv_rn(amax, 448.0f);
  g.rcp = __frcp_rn(g.scale);
  return g;
}

// x / scale for a scale whose correctly rounded reciprocal r is at hand: q = x r, then q + (x - q scale) r, the remainder
// exact by FMA.  Correctly rounded by Markstein's theorem (IBM J. Res. Dev. 34, 1990) wherever nothing underflows, at a
// third of the instructions of a division; quotients that could underflow are far below the smallest code.
__device__ __forceinline__ float div_by(float x, float scale, float r) {
  const float q = x * r;
  return fmaf(fmaf(-q, scale, x), r, q);
}

// Four values over one scale as e4m3 codes, nearest even, clamped to +-448 (NaN stays NaN).  Over a power of two the
// product with the reciprocal is exact already.
template <bool kPow2>
__device__ __forceinline__ uint32_t quant_e4m3x4(float a, float b, float c, float d, GroupScale g) {
  auto over = [&](float x) { return kPow2 ? x * g.rcp : div_by(x, g.scale, g.rcp); };
  const __nv_fp8x2_storage_t lo = __nv_cvt_float2_to_fp8x2(make_float2(over(a), over(b)), __NV_SATFINITE, __NV_E4M3);
  const __nv_fp8x2_storage_t hi = __nv_cvt_float2_to_fp8x2(make_float2(over(c), over(d)), __NV_SATFINITE, __NV_E4M3);
  return static_cast<uint32_t>(lo) | (static_cast<uint32_t>(hi) << 16);
}

// Four codes times their scale as bf16 pairs.  The codes widen to fp16 exactly; the product is rounded to bf16 once,
// and not at all when the scale is a power of two (four significant bits).
__device__ __forceinline__ void dequant_e4m3x4(uint32_t codes, float scale, uint32_t& lo, uint32_t& hi) {
  const __half2_raw h0 = __nv_cvt_fp8x2_to_halfraw2(static_cast<__nv_fp8x2_storage_t>(codes & 0xffffu), __NV_E4M3);
  const __half2_raw h1 = __nv_cvt_fp8x2_to_halfraw2(static_cast<__nv_fp8x2_storage_t>(codes >> 16), __NV_E4M3);
  const float2 f0 = __half22float2(__half2(h0)), f1 = __half22float2(__half2(h1));
  const __nv_bfloat162 b0 = __floats2bfloat162_rn(f0.x * scale, f0.y * scale);
  const __nv_bfloat162 b1 = __floats2bfloat162_rn(f1.x * scale, f1.y * scale);
  lo = *reinterpret_cast<const uint32_t*>(&b0);
  hi = *reinterpret_cast<const uint32_t*>(&b1);
}

}  // namespace b200dsa
