// The MFMA decode kernels (decode_stream.hpp) of caches with a scale for each block and head.
//
// A tile of 32 tokens is two blocks, and the QK^T product leaves a lane the scores
// of 8 tokens of one of them: its K scale multiplies them, its V scale their
// weights ahead of the product with V.  Two 4-byte loads a lane and tile, and 8
// multiplications.
#include "decode_stream.hpp"

namespace cf {

namespace {

template <int KT>
int32_t launch_kt(const DecodeBlockParams& p, int q_dt, hipStream_t stream) {
  if (q_dt == kF32) return launch_d<kF32, KT>(p, stream);
  return q_dt == kF16 ? launch_d<kF16, KT>(p, stream) : launch_d<kBF16, KT>(p, stream);
}

}  // namespace

int32_t launch_decode_mfma(const DecodeBlockParams& p, int q_dt, int kv_dt, hipStream_t stream) {
  return kv_dt == kI8 ? launch_kt<kI8>(p, q_dt, stream) : launch_kt<kE4M3>(p, q_dt, stream);
}

}  // namespace cf
