// Device helpers of the dense products, their checkpoints and gradients:
// activations, e4m3 / e8m0 conversion.
//
// An 8-bit checkpoint keeps a row in blocks of 128 values: e4m3 bytes and one
// e8m0 scale per block, a power of two 2^e with the least e for which
// amax <= 448 * 2^e (and e >= -117). Scaling by a power of two is exact, so the
// only rounding is the e4m3 one (half a step: 2^-4 relative above the
// subnormals), and every restored value q * 2^e (four significant bits, least
// magnitude 2^-126) is a bf16 number: the backward's bf16 matrix products see
// the checkpoint exactly. In a block of the largest scale, 2^120, magnitudes are
// held at 240 * 2^120 (256 * 2^120 would be infinite). A block holding an infinity or NaN gets the e8m0 NaN
// code and comes back as NaN throughout.
#pragma once

#include "moe_common.cuh"
#include "train_kernels.h"

namespace moe {

constexpr int kMinScaleExp = -117;

// e8m0 code of a block from its largest magnitude (bits of a non-negative
// float; NaN and infinity compare above every finite value as integers).
__device__ __forceinline__ uint32_t e8m0_of_amax(uint32_t amax_bits) {
  if (amax_bits >= 0x7f800000u) return 255u;
  // amax = 1.f * 2^p: 448 = 1.75 * 2^8, so e = p - 8 while the significand is at most 1.75
  const int p = (int)(amax_bits >> 23) - 127;
  const int e = p - ((amax_bits & 0x7fffffu) <= 0x600000u ? 8 : 7);
  return (uint32_t)((e < kMinScaleExp ? kMinScaleExp : e) + 127);
}
// Scaled values of a block, held below infinity (a rare, block-uniform branch).
constexpr uint32_t kTopScaleCode = 120 + 127;
__device__ __forceinline__ float hold_finite(float v) { return fminf(fmaxf(v, -240.f), 240.f); }
// 2^-e for a code made above (e in [-117, 120]); NaN for the NaN code.
__device__ __forceinline__ float e8m0_inverse(uint32_t code) {
  return code == 255u ? __uint_as_float(0x7fffffffu) : __uint_as_float((254u - code) << 23);
}
// 2^e for any code a caller may hand over.
__device__ __forceinline__ float e8m0_value(uint32_t code) {
  return code == 255u ? __uint_as_float(0x7fffffffu) : __uint_as_float(code ? code << 23 : 0x00400000u);
}

__device__ __forceinline__ uint32_t e4m3x4(float a, float b, float c, float d) {
  const __nv_fp8x2_storage_t lo = __nv_cvt_float2_to_fp8x2(make_float2(a, b), __NV_SATFINITE, __NV_E4M3);
  const __nv_fp8x2_storage_t hi = __nv_cvt_float2_to_fp8x2(make_float2(c, d), __NV_SATFINITE, __NV_E4M3);
  return (uint32_t)lo | ((uint32_t)hi << 16);
}
__device__ __forceinline__ float2 e4m3x2_value(uint32_t v16) {
  const __half2_raw h = __nv_cvt_fp8x2_to_halfraw2((__nv_fp8x2_storage_t)v16, __NV_E4M3);
  return __half22float2(*reinterpret_cast<const __half2*>(&h));
}
__device__ __forceinline__ float e4m3_value(uint8_t v) { return e4m3x2_value(v).x; }

__device__ __forceinline__ uint32_t pack_bf16(float a, float b) {
  const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
  return *reinterpret_cast<const uint32_t*>(&h);
}
__device__ __forceinline__ float2 unpack_bf16(uint32_t v) {
  return __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(&v));
}

// Read-only load through L1, or through L2 alone in an early launch (train_kernels.h).
template <bool EARLY, typename T>
__device__ __forceinline__ T load_input(const T* p) {
  return EARLY ? __ldcg(p) : __ldg(p);
}
// Elements `at`, at + 1 of a row of 16-bit values, which start at an even address;
// those outside [begin, end) are 0 and not read.
template <bool EARLY>
__device__ __forceinline__ uint32_t load_pair(const uint16_t* row, int at, int begin, int end) {
  if (at >= begin && at + 1 < end) return load_input<EARLY>(reinterpret_cast<const uint32_t*>(row + at));
  uint32_t v = 0;
  if (at >= begin && at < end) v = load_input<EARLY>(row + at);
  if (at + 1 >= begin && at + 1 < end) v |= (uint32_t)load_input<EARLY>(row + at + 1) << 16;
  return v;
}

__device__ __forceinline__ float sigmoid_f(float z) { return 1.0f / (1.0f + expf(-z)); }

// 1 / (1 + e^-z) with the hardware exponential and reciprocal.
__device__ __forceinline__ float sigmoid_fast(float z) { return __fdividef(1.0f, 1.0f + __expf(-z)); }

// Phi(z), good to z^2 + 8 units of 2^-23 of itself down to the least normal number: as 1 + erf(z / sqrt 2) the lower
// tail cancels (4 % off at z = -5, zero below -5.6). With a = |z| and t = 1 / (1 + 0.3 a), e^(a^2 / 2) Phi(-a) is t times
// a smooth function of t on (0, 1]; the polynomial is its least relative maximum error of degree 7 (1.5e-7), fitted by
// Lawson's reweighted least squares in 64 bits for a up to 14. FAST: the hardware exponential (another z^2 / 2 units),
// for results in bf16. gelu of 4096 x 7168 values, K = 256: 53 us in bf16, 56 with erff, 92 with erfcf.
template <bool FAST>
__device__ __forceinline__ float normal_cdf(float z) {
  const float a = fabsf(z), t = __fdividef(1.0f, fmaf(0.3f, a, 1.0f));
  float p = 0.0356747732f;
  p = fmaf(p, t, -0.157203078f);
  p = fmaf(p, t, 0.20635349f);
  p = fmaf(p, t, -0.05368363f);
  p = fmaf(p, t, 0.12856162f);
  p = fmaf(p, t, 0.09991349f);
  p = fmaf(p, t, 0.12075396f);
  p = fmaf(p, t, 0.1196293f);
  const float e = -0.5f * z * z, q = p * t * (FAST ? __expf(e) : expf(e));      // Phi(-a); NaN stays
  return z > 0.f ? 1.0f - q : q;
}

// Single-input activations (codes 0..3); SwiGLU is first * silu(second).
__device__ __forceinline__ float act_value(float z, int act) {
  switch (act) {
    case kActRelu: return z < 0.f ? 0.f : z;              // NaN stays
    case kActGelu: return z * normal_cdf<false>(z);
    case kActSilu: return z / (1.0f + expf(-z));
    default: return z;
  }
}
template <bool FAST>
__device__ __forceinline__ float act_slope(float z, int act) {
  switch (act) {
    case kActRelu: return z > 0.f ? 1.f : z <= 0.f ? 0.f : z;      // NaN stays, as in the value
    case kActGelu:
      return normal_cdf<FAST>(z) + z * 0.39894228040143268f * (FAST ? __expf(-0.5f * z * z) : expf(-0.5f * z * z));
    case kActSilu: {
      const float s = FAST ? sigmoid_fast(z) : sigmoid_f(z);
      return s * (1.0f + z * (1.0f - s));
    }
    default: return 1.f;
  }
}

}  // namespace moe
