// Parameters shared by the paged-decode kernels and their host launchers.
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

namespace cf {

// All strides are in elements of the tensor they index.
struct DecodeParams {
  const void* q;
  int64_t q_sb, q_sh;  // q [B, Hq, D], D stride 1
  const void* k;
  const void* v;
  int64_t k_s[4];  // k_cache [NB, bs, Hkv, D]
  int64_t v_s[4];  // v_cache [NB, bs, Hkv, D]
  const int32_t* tables;
  int64_t t_sb, t_sm;  // block_tables [B, Mb]
  const int32_t* seq_lens;
  int64_t sl_s;  // seq_lens [B]
  const int32_t* shared;  // optional [B]: leading tokens sequence b shares with b - 1
  int64_t sh_s;
  const float* k_scale;
  const float* v_scale;
  int64_t ks_s, vs_s;  // 0 when the scale is a single value
  void* out;
  int64_t o_sb, o_sh;  // out [B, Hq, D], D stride 1
  float* ws_o;         // generic path: [B, Hq, max_parts, D] un-normalized partial outputs;
                       // MFMA path: [rows, D] partial rows (see decode_mfma.hip)
  float* ws_ml;        // running max and sum per partial row
  int2* own_desc;      // MFMA path: per (sequence, KV head), the sequence's own run
  int2* pre_desc;      // MFMA path: per (sequence, KV head), its shared-prefix run
  int64_t rec_own;     // MFMA path: first row of the per-(sequence, head) own-run records
  int64_t rec_pre;     // ... and of the shared-prefix records
  float scale;
  int B, Hq, Hkv, G, D, bs, Mb, PT, max_parts;
  int NB;  // cache blocks; a block id outside [0, NB) contributes no tokens
};

// A decode call over a cache with a scale for each block and head.
struct DecodeBlockParams : DecodeParams {
  int64_t ks_b, vs_b;  // strides over blocks of k_scale and v_scale [NB, Hkv] (ks_s, vs_s: over heads)
};

// A decode call that also accounts for the weights: the kernels leave every
// score and the rows' final (m, l), from which decode_weights_kernel forms them.
struct DecodeWeightsParams : DecodeParams {
  float* ws_s;    // scores [B, Hkv, s_cap / 32, 2, G, 16]: log2 units (MFMA path) or natural ones, -inf where masked
  float* ws_fin;  // [B, Hq, 2] final reference and sum of a row
  int64_t s_cap;  // tokens of a score row, a multiple of 32
  float* weights;  // [B, Hw, >= Mb * bs] f32, last stride 1
  int64_t w_sb, w_sh;
  int Hw;  // Hkv, or 1
  float decay;
};

// Workgroups that form the accounts, 1,024 tokens each.
inline int64_t account_blocks(const DecodeWeightsParams& p) {
  return ((int64_t)p.Mb * p.bs + 1023) / 1024 * p.B * p.Hw;
}
// Accounts of one KV head each are formed in the launch that joins the rows, if
// they are few: the joining kernel's registers leave fewer waves to hide the
// scores' latency.  4 requests of 512 f32 tokens: 4.1 us against 4.3 and 4.0 in
// two launches; 29 sequences of 2,928 tokens (696 workgroups) 7.3 against 4.4 and
// 4.4; 79 of 1,073 (1,264) 9.0 against 4.2 and 5.5; 64 of 8,192 (4,096) 22.6
// against 4.3 and 13.8.
inline bool accounts_with_rows(const DecodeWeightsParams& p) { return p.Hw == p.Hkv && account_blocks(p) <= 1024; }
inline bool accounts_aligned(const DecodeWeightsParams& p) {
  return ((uintptr_t)p.weights & 15) == 0 && p.w_sb % 4 == 0 && p.w_sh % 4 == 0;
}

// Where a token's score lies among its tile's 32 * G: 16 floats a query head,
// those of tokens 8 i .. 8 i + 3 in the first half and of 8 i + 4 .. 8 i + 7 in
// the second.  A wave of the streaming kernel holds tokens 8 (lane / 16) + 4 x
// .. + 3 of its heads, so each of its two stores fills whole lines.
__device__ __forceinline__ int64_t score_at(int t, int g, int G) {
  return (int64_t)(t >> 5) * (32 * G) + (((t >> 2) & 1) * 16 * G + g * 16 + ((t >> 3) & 3) * 4 + (t & 3));
}

// Launchers (return a CF_* status; kernels are enqueued on `stream`).
int32_t launch_decode_generic(const DecodeParams& p, int q_dt, int kv_dt, hipStream_t stream);
int32_t launch_decode_mfma(const DecodeParams& p, int q_dt, int kv_dt, hipStream_t stream);
int32_t launch_decode_generic(const DecodeBlockParams& p, int q_dt, int kv_dt, hipStream_t stream);
int32_t launch_decode_mfma(const DecodeBlockParams& p, int q_dt, int kv_dt, hipStream_t stream);
// The same with scores and final (m, l) written (the call is one that the
// plain launcher takes), and the accounts formed from them.
int32_t launch_decode_generic(const DecodeWeightsParams& p, int q_dt, int kv_dt, hipStream_t stream);
int32_t launch_decode_mfma(const DecodeWeightsParams& p, int q_dt, int kv_dt, hipStream_t stream);
int32_t launch_decode_weights(const DecodeWeightsParams& p, bool log2_units, hipStream_t stream);
bool decode_mfma_supported(const DecodeParams& p, int q_dt, int kv_dt);
// Whether its scales' offsets are what the MFMA kernel takes (32 bits).
bool decode_mfma_block_scales(const DecodeBlockParams& p);
// Workspace of the MFMA path: two (m, l, o) partial slots per launched wave.
uint64_t decode_mfma_workspace_bytes(int64_t batch, int64_t num_q_heads, int64_t num_kv_heads, int64_t head_dim);
void decode_mfma_bind_workspace(DecodeParams& p, void* workspace);

int32_t launch_decode_reduce(const DecodeParams& p, int q_dt, hipStream_t stream);
int32_t launch_decode_reduce(const DecodeWeightsParams& p, int q_dt, hipStream_t stream);
// LDS bytes of one generic-kernel workgroup (G query heads, partition PT).
size_t generic_lds_bytes(int64_t G, int64_t D, int64_t PT, int64_t bs);

}  // namespace cf
