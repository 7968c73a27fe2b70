// Rows of a cache held in 4 bits: groups of 32 channels with a scale each
// (include/flash_prologue.h has the format), written by the lanes of gqa_fwd.cu.
//
// A word of a row holds 8 channels, and word w belongs to group w % (D / 32). A
// lane of the prologue owns 8 channels of either half of the row, words c and
// c + L (L = D / 16 lanes a row), which are in one group; its other half is the
// lane L / 2 away. So a group's extremes are 16 values of a lane and one shuffle.
#pragma once

#include "prologue_common.cuh"

namespace flash_prologue {

__device__ __forceinline__ float max_or_nan(float a, float b) {
  float y;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(y) : "f"(a), "f"(b));
  return y;
}

// -1/8 of the value of largest magnitude, cut to five significant bits: with |code|
// at most 8 every s * code has eight, so the 16-bit kernels can use it unrounded.
// NaN where the group holds an infinity or NaN.
template <typename T>
__device__ __forceinline__ float int4_scale(float high, float low) {
  float s = -0.125f * (high >= -low ? high : low);
  s = __int_as_float(__float_as_int(s) & ~0x7ffff);
  constexpr bool kHalf = std::is_same<T, __half>::value;
  // FP16: s * code inside its range, and no bit of it below 2^-24. BF16: 1 / s and 24 s are normal numbers.
  const float size = fminf(fmaxf(fabsf(s), kHalf ? 0x1p-20f : 0x1p-100f), kHalf ? 7936.f : 0x1p122f);
  const float kept = s == 0.f ? 0.f : copysignf(size, s);
  return high - high == 0.f && low - low == 0.f ? kept : __int_as_float(0x7fc00000);
}

// The word of eight channels a[0].x, a[0].y, ..., a[3].y: code(x) = clamp(rint(x / s), -8, 7) + 8.
// inv is 1 / s correctly rounded; with it, q + (x - q s) inv of q = x inv rounds to the
// quotient that a division gives (Markstein's theorem), so codes do not depend on how it is done.
__device__ __forceinline__ uint32_t int4_word(const float2 (&a)[kPairs], float s, float inv) {
  uint32_t word = 0;
#pragma unroll
  for (int p = 0; p < kPairs; ++p) {
    float2 q = __fmul2_rn(a[p], splat2(inv));
    const float2 rest = __ffma2_rn(q, splat2(-s), a[p]);
    q = __ffma2_rn(rest, splat2(inv), q);
    q.x = fminf(fmaxf(q.x, -8.f), 7.f);
    q.y = fminf(fmaxf(q.y, -8.f), 7.f);
    // 1.5 * 2^23 + 8: the sum is rounded to a whole number (ties to even), whose low bits are the code.
    q = __fadd2_rn(q, splat2(12582920.f));
    const uint32_t both = __byte_perm(__float_as_uint(q.x), __float_as_uint(q.y), 0x5410);
    word |= (both & 0x000f000fu) << (4 * p);
  }
  return word;
}

// A lane's two words and its group's scale of a row that L lanes hold, lane c of them this one.
template <typename T, int L>
__device__ __forceinline__ void int4_encode(const float2 (&a)[kPairs], const float2 (&b)[kPairs], uint32_t& wa,
                                            uint32_t& wb, uint16_t& scale) {
  float high = a[0].x, low = a[0].x;
#pragma unroll
  for (int p = 0; p < kPairs; ++p) {
    high = max_or_nan(max_or_nan(high, max_or_nan(a[p].x, a[p].y)), max_or_nan(b[p].x, b[p].y));
    low = fminf(fminf(low, fminf(a[p].x, a[p].y)), fminf(b[p].x, b[p].y));
  }
  high = max_or_nan(high, __shfl_xor_sync(0xffffffffu, high, L / 2));
  low = fminf(low, __shfl_xor_sync(0xffffffffu, low, L / 2));
  const float s = int4_scale<T>(high, low);
  scale = (uint16_t)(__float_as_uint(s) >> 16);
  if (s == s) {
    const float inv = s == 0.f ? 0.f : __frcp_rn(s);
    wa = int4_word(a, s, inv);
    wb = int4_word(b, s, inv);
  } else {
    wa = wb = 0x88888888u;
  }
}

}  // namespace flash_prologue
