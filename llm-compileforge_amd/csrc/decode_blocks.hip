// The MFMA decode kernels (decode_stream.hpp) of caches with a scale for each block and head.
//
// A tile of 32 tokens is two blocks, and the QK^T product leaves a lane the scores
// of 8 tokens of one of them: its K scale multiplies them, its V scale their
// weights ahead of the product with V: two 4-byte loads a lane and tile, 8
// multiplications, and P in two bf16 terms.  Bound by HBM as the kernel with a scale
// a head: 64 sequences of 1,024 to 8,192 tokens, half of them on a shared prefix
// (528 MB, e4m3 under bf16, 32 / 8 heads of 128), 96 us (5.5 TB/s) against 93 with one
// scale a head; 48 sequences of int8 under fp16 (456 MB) 84 us.  int8 under bf16 takes
// 12 instructions for 8 codes where e4m3 takes 4 and int8 under fp16 10, and is bound
// by them: 99 us for the first batch.  The scales are loaded ahead of the tile's rows,
// by offsets of 32 bits: behind them they took 132.
#include <algorithm>

#include "decode_stream.hpp"

namespace cf {

namespace {

template <int KT>
int32_t launch_kt(const DecodeBlockParams& p, int q_dt, hipStream_t stream) {
  if (q_dt == kF32) return launch_d<kF32, KT>(p, stream);
  return q_dt == kF16 ? launch_d<kF16, KT>(p, stream) : launch_d<kBF16, KT>(p, stream);
}

}  // namespace

bool decode_mfma_block_scales(const DecodeBlockParams& p) {
  const int64_t most = std::max((p.NB - 1) * p.ks_b + (p.Hkv - 1) * p.ks_s, (p.NB - 1) * p.vs_b + (p.Hkv - 1) * p.vs_s);
  return most < ((int64_t)1 << 31);
}

int32_t launch_decode_mfma(const DecodeBlockParams& p, int q_dt, int kv_dt, hipStream_t stream) {
  if (!decode_mfma_block_scales(p)) {
    set_error("decode: block scales whose offsets pass 31 bits");
    return CF_ERR_UNSUPPORTED;
  }
  return kv_dt == kI8 ? launch_kt<kI8>(p, q_dt, stream) : launch_kt<kE4M3>(p, q_dt, stream);
}

}  // namespace cf
