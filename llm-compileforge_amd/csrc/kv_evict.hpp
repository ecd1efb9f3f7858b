// Eviction from a paged cache by accumulated attention weight: which tokens
// each head keeps, and the moves that close the holes.
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

namespace cf {

// All strides are in elements.
struct EvictSelectParams {
  const float* weights;  // [B, H, S], S stride 1
  int64_t w_sb, w_sh;
  const int32_t* lens;  // [B]
  int64_t l_s;
  const int32_t* positions;  // [B, H, S], S stride 1, or null: a slot's index is its position
  int64_t p_sb, p_sh;
  const int32_t* kept;  // [B]: slots that have an entry in positions
  const int32_t* seen;  // [B]: tokens of the sequence so far, evicted ones included
  int64_t kept_s, seen_s;
  int32_t* keep;  // [B, H, budget], budget stride 1
  int64_t k_sb, k_sh;
  int32_t* new_lens;  // [B]
  int64_t n_s;
  int B, H, S, budget, sink, recent;
};

struct EvictMoveParams {
  const int32_t* keep;  // [B, Hw, budget], budget stride 1
  int64_t k_sb, k_sh;
  const int32_t* lens;  // [B]
  int64_t l_s;
  const int32_t* tables;  // [B, Mb]
  int64_t t_sb, t_sm;
  void* cache[2];  // K, V [NB, bs, Hkv, D]
  int64_t c_s[2][4];
  float* weights;  // [B, Hw, S], S stride 1, or null
  int64_t w_sb, w_sh;
  int32_t* positions;  // [B, Hw, S], S stride 1, or null
  int64_t p_sb, p_sh;
  const int32_t* kept;
  const int32_t* seen;
  int64_t kept_s, seen_s;
  int64_t NB;
  int B, Hw, Hkv, D, bs, Mb, S, budget;
  int mode[2];  // how K and V rows move; set by the launcher
};

int32_t launch_evict_select(const EvictSelectParams& p, hipStream_t stream);
int32_t launch_evict_move(const EvictMoveParams& p, int elem_bytes, hipStream_t stream);

}  // namespace cf
