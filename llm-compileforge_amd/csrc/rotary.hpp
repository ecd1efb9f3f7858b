// Rotary positions of one or several axes on query and key rows, with the key
// and value rows written to their paged slots.
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

namespace cf {

constexpr int kMaxRotaryAxes = 4;

// All strides are in elements.
struct RotaryParams {
  const void* x[3];  // queries, keys, values [T, H, D]; no keys and values if Hkv == 0
  int64_t x_s[3][3];
  void* out;  // rotated queries [T, Hq, D]
  int64_t o_s[3];
  void* cache[2];  // K, V [NB, bs, Hkv, D]
  int64_t c_s[2][4];
  const float* scale[2];  // e4m3fn caches: [Hkv] or [1]
  int64_t sc_s[2];        // 0 for a single scale
  const void* slots;      // [T] i32 | i64: block * bs + offset
  int64_t slot_s;
  const void* positions;  // [axes, T] i32 | i64
  int64_t p_sa, p_st;
  const float* inv_freq;  // [pairs]
  int64_t f_s;
  int64_t NB, T;
  float rotary_scale;
  int Hq, Hkv, D, bs, pairs, axes;
  int section[kMaxRotaryAxes];  // pairs of each axis
  bool cycled, adjacent, pos64, slot64;
  // set by the launcher: which of queries, keys and values move in whole
  // pieces, and whether values go through the transposing stage
  bool vec[3], v_tile;
};

int32_t launch_rotary(RotaryParams p, int x_dt, int cache_dt, hipStream_t stream);

}  // namespace cf
