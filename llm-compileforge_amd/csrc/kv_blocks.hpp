// New K and V rows into paged caches with a scale for each block and head.
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

namespace cf {

// All strides are in elements; index 0: keys, 1: values.
struct KvBlocksParams {
  const void* x[2];  // new rows [T, H, D]
  int64_t x_s[2][3];
  void* cache[2];  // [NB, bs, H, D]
  int64_t c_s[2][4];
  float* scale[2];  // [NB, H]
  int64_t s_s[2][2];
  const int32_t* tables;  // [N, Mb]
  int64_t t_sn, t_sm;
  const int32_t* lens;  // [N]: tokens of a sequence, the new rows included
  int64_t l_s;
  const int32_t* start;  // [N + 1]: first row of each sequence; null: row n is sequence n's
  int64_t st_s;
  int64_t T, NB, units;  // units: an upper bound on the blocks written to
  int N, Mb, H, D, bs;
};

int32_t launch_kv_blocks(KvBlocksParams p, int x_dt, int cache_dt, hipStream_t stream);

}  // namespace cf
