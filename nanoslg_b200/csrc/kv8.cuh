// The 8-bit KV cache format, shared by the kernels that write and read it.
//
// One layer: e4m3 codes [num_pages, num_kv_heads, page_size, head_dim] for K and for V and
// one fp32 scale per block, [num_pages, num_kv_heads]; a block is the page_size tokens of
// one page for one kv head, contiguous in memory (2 KiB at page_size 16, head_dim 128).
// value = code * scale. The writer's scale is a power of two: the smallest s with
// amax <= 448 * s, so a code keeps e4m3's four significant bits whatever the block's
// magnitude (a float format gains nothing from a finer scale), dividing by it is exact,
// and when a later token makes the block's scale grow, re-rounding the older codes moves
// their exponents exactly: only codes that fall into e4m3's subnormals are rounded again.
// Scale 0: a block of zeros. Scale NaN: the block holds a value that is not finite, and
// all of it reads as NaN.
#pragma once

#include "common.cuh"

namespace nslg {

// Codes of two values (lo in the low byte), nearest even, saturating; NaN stays NaN.
__device__ __forceinline__ uint16_t e4m3x2_from_f32(float lo, float hi) {
  uint16_t r;
  asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(r) : "f"(hi), "f"(lo));
  return r;
}

// Two codes as f16x2 (exact: every e4m3 value is an f16 value).
__device__ __forceinline__ uint32_t f16x2_from_e4m3x2(uint16_t c) {
  uint32_t r;
  asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(r) : "h"(c));
  return r;
}

__device__ __forceinline__ float2 f32x2_from_e4m3x2(uint16_t c) {
  const uint32_t h = f16x2_from_e4m3x2(c);
  return __half22float2(*reinterpret_cast<const __half2*>(&h));
}

// |x| as an unsigned word: ordered like the magnitudes, infinities and NaN above all.
__device__ __forceinline__ uint32_t abs_bits(float x) { return __float_as_uint(x) & 0x7FFFFFFFu; }

// The scale of a block whose largest magnitude has these bits. 448 = 1.75 * 2^8: the
// exponent is the magnitude's minus 8, one more where its significand is above 1.75.
// Never below 2^-126 (1 / scale stays finite).
__device__ __forceinline__ float scale_from_amax(uint32_t bits) {
  if (bits == 0u) return 0.f;
  if (bits >= 0x7F800000u) return __uint_as_float(0x7FC00000u);
  const int e = static_cast<int>((bits + 0x1FFFFFu) >> 23) - 8;
  return __uint_as_float(static_cast<uint32_t>(e < 1 ? 1 : e) << 23);
}

// The tensor-core readers take V's scale as a power of two in the exponent of a weight, and its
// inverse in the row's sum, which must not overflow: a V block of a smaller scale than this
// counts as zeros there (values below 448 * 2^-100).
constexpr float kLeastE = -100.f;
// A block of zeros in V (or of a scale below 2^-100, or NaN) has no exponent, only a part in the
// row's sum l. Behind blocks that have one it takes one kZeroE below theirs, so that the running
// maximum M follows it only where it outweighs them by 2^60. Before any it takes 0: M and l are
// those of the plain scores, and the first block with an exponent sets M anew, whatever its
// magnitude, but not by more than kMostDown downwards: l, at most 2^8 a position until then, is
// multiplied by 2^kMostDown at most, and a row whose weights lie further below a block of zeros
// is less than 448 * 2^-90.
constexpr float kZeroE = 60.f;
constexpr float kMostDown = 90.f;
__device__ __forceinline__ bool has_exponent(float scale) {
  return scale >= 7.888609052210118e-31f && scale < INFINITY;   // 2^-100; not NaN
}

// The larger of two scales; NaN wins.
__device__ __forceinline__ float scale_max(float a, float b) {
  return (a != a || b != b) ? __uint_as_float(0x7FC00000u) : fmaxf(a, b);
}

// What a value is multiplied with before it is rounded to a code of a block of this scale.
__device__ __forceinline__ float scale_inverse(float s) { return s == 0.f ? 0.f : 1.f / s; }

// Two codes of a block of scale `was`, rounded again for the scale `now` (ratio = was / now).
__device__ __forceinline__ uint16_t e4m3x2_rescale(uint16_t c, float ratio) {
  const float2 v = f32x2_from_e4m3x2(c);
  return e4m3x2_from_f32(v.x * ratio, v.y * ratio);
}

// A cache value in the activation type: rounded once; a finite value beyond fp16's range
// (65504 rounds up to the code of 65536) saturates instead of becoming an infinity.
template <typename T>
__device__ __forceinline__ T from_cache(float x) {
  return Elem<T>::from_f(x);
}
template <>
__device__ __forceinline__ __half from_cache<__half>(float x) {
  const float a = fabsf(x);
  return __float2half_rn(a > 65504.f && a < INFINITY ? copysignf(65504.f, x) : x);
}

}  // namespace nslg
