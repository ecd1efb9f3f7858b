// Caches in 8 bits with a scale for each block of tokens and KV head: the value
// of code c of block b and head h is c * scale[b][h].  Codes are e4m3fn (up to
// 448 in magnitude) or int8 (up to 127).
//
// The scale of a block that holds values up to amax is the least that its codes
// can reach them with: amax / 127 for int8, and for e4m3fn the next power of two
// from amax / 448 on (quotients as products with the rounded reciprocal).  A
// floating-point code loses no precision by it (its steps are relative; the
// smallest normal one is 2^14 below amax in either case), the division by it is exact, and where a later row widens the block's scale, the
// codes already there move by whole exponents and are exact still, unless they
// fall below the smallest normal one.  int8 codes are rounded again by a widening,
// by half a step of the new scale at most.
#pragma once

#include "cf_device.hpp"
#include "mfma_tile.hpp"

namespace cf {
namespace {

constexpr float kLeastScale = 9.094947017729282e-13f;  // 2^-40: that of zeros alone

// The least scale for values of magnitude bits `amax` (NaN above infinity above
// the numbers).  Where one is not finite no scale reaches it: NaN, with which
// every value of the block reads as NaN.
template <int CT>
__device__ __forceinline__ float least_scale(uint32_t amax) {
  if (amax >= 0x7F800000u) return u2f(0x7FC00000u);
  if constexpr (CT == kI8) {
    return fmaxf(u2f(amax) * (1.0f / 127.0f), kLeastScale);
  } else {
    const uint32_t a = f2u(fmaxf(u2f(amax) * (1.0f / 448.0f), kLeastScale));
    return u2f((a + 0x7FFFFFu) & 0x7F800000u);
  }
}

// The scale of a block that had `old` (0: it starts anew) and takes rows that
// need `least`; a NaN of either stays.
__device__ __forceinline__ float widened(float old, float least) {
  return old != old || least != least ? u2f(0x7FC00000u) : fmaxf(old, least);
}

// x / scale as a code, the division rounded as torch's; int8 codes round to the
// nearest integer, ties to even (0 under a NaN).
template <int CT>
__device__ __forceinline__ uint8_t block_code(float x, float scale) {
  const float q = x / scale;
  if constexpr (CT == kI8) {
    return (uint8_t)(int8_t)(q == q ? (int)__builtin_rintf(fminf(fmaxf(q, -127.0f), 127.0f)) : 0);
  } else {
    return e4m3_from_f32(q);
  }
}

}  // namespace
}  // namespace cf
