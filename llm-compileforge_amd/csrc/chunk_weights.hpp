// Accounts of prompt chunks: the attention weight that the rows of a chunk put
// on each cached token.
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

namespace cf {

// All strides are in elements.
struct ChunkWeightsParams {
  const void* q;  // [Tq, Hq, D], D stride 1
  int64_t q_sr, q_sh;
  const void* k;  // k_cache [NB, 16, Hkv, D], D stride 1
  int64_t k_s[4];
  const int32_t* tables;  // [N, Mb]
  int64_t t_sb, t_sm;
  const int32_t* seq_lens;  // [N]
  int64_t sl_s;
  const int32_t* q_start;  // [N + 1]
  int64_t qs_s;
  const float* k_scale;  // [Hkv] or [1] (e4m3fn), else null
  int64_t ks_s;          // 0 for a single scale
  float* weights;        // [N, Hw, >= Mb * 16], last stride 1
  int64_t w_sb, w_sh;
  float scale, decay;
  int observe;  // last rows of a chunk that count; 0: all of them
  int N, Tq, Hq, Hkv, Hw, G, D, Mb, NB;
  // set by chunk_weights_bind_workspace
  float2* ws_ml;  // [ml_pieces, stat_rows, Hq] (reference, sum) of a row over a run of its tokens
  float* ws_p;    // [pieces, Hkv, Mb * 16] sums over a run of columns
  int* ws_np;     // [stat_rows] runs of the row's tokens
  int* ws_tp;     // [N, blocks of 256 tokens] runs of the block's columns
  int64_t stat_rows;
  bool compact;   // rows and pieces are numbered by the chunk's observers
  bool joined;    // the rows' runs are joined before the tokens kernel
  int ml_pieces;
  int row_steps, col_steps;  // steps that a workgroup takes at least
  int piece_rows;            // rows of col_steps steps
};

bool chunk_weights_supported(const ChunkWeightsParams& p, int q_dt, int k_dt);
// Workspace of a call; chunk_weights_bind_workspace lays it out.
uint64_t chunk_weights_workspace_bytes(int64_t num_q_tokens, int64_t num_chunks, int64_t num_q_heads,
                                       int64_t num_kv_heads, int64_t max_blocks, int64_t observe);
void chunk_weights_bind_workspace(ChunkWeightsParams& p, void* workspace);
int32_t launch_chunk_weights(const ChunkWeightsParams& p, int q_dt, int k_dt, hipStream_t stream);

}  // namespace cf
