// The MFMA decode kernels (decode_stream.hpp) of caches with a scale for each KV head, or none: launchers, their
// workspace and what they take.
#include "decode_stream.hpp"

namespace cf {

namespace {

bool aligned16(const void* ptr) { return ((uintptr_t)ptr & 15) == 0; }

// Workspace layout: [partial rows: o, D f32 each, 256-byte padded]
// [(m, l) per row, padded] [own-run descriptors: int2 per (sequence, KV
// head), padded] [prefix descriptors, same].  Rows: 2 slots x 16 columns per
// wave, then G own-run and G prefix records per (sequence, KV head).
uint64_t stream_waves() { return (uint64_t)cu_count() * kStreamBlocksPerCU * 4; }
uint64_t pad256(uint64_t x) { return (x + 255) & ~(uint64_t)255; }
uint64_t slot_rows() { return stream_waves() * 2 * kSlotCols; }
uint64_t total_rows(int64_t batch, int64_t num_q_heads) { return slot_rows() + 2 * (uint64_t)batch * num_q_heads; }

template <class P>
int32_t launch_any(const P& p, int q_dt, int kv_dt, hipStream_t stream) {
  if (q_dt == kF16) return kv_dt == kE4M3 ? launch_d<kF16, kE4M3>(p, stream) : launch_d<kF16, kF16>(p, stream);
  if (q_dt == kF32 && kv_dt == kF32) return launch_d<kF32, kF32>(p, stream);
  if (q_dt == kF32) return kv_dt == kE4M3 ? launch_d<kF32, kE4M3>(p, stream) : launch_d<kF32, kBF16>(p, stream);
  return kv_dt == kE4M3 ? launch_d<kBF16, kE4M3>(p, stream) : launch_d<kBF16, kBF16>(p, stream);
}

}  // namespace

uint64_t decode_mfma_workspace_bytes(int64_t batch, int64_t num_q_heads, int64_t num_kv_heads, int64_t head_dim) {
  const uint64_t rows = total_rows(batch, num_q_heads);
  const uint64_t desc = pad256((uint64_t)batch * num_kv_heads * 8);
  return pad256(rows * head_dim * 4) + pad256(rows * 2 * 4) + 2 * desc;
}

void decode_mfma_bind_workspace(DecodeParams& p, void* workspace) {
  const uint64_t rows = total_rows(p.B, p.Hq);
  const uint64_t desc = pad256((uint64_t)p.B * p.Hkv * 8);
  char* w = (char*)workspace;
  p.ws_o = (float*)w;
  w += pad256(rows * p.D * 4);
  p.ws_ml = (float*)w;
  w += pad256(rows * 2 * 4);
  p.own_desc = (int2*)w;
  w += desc;
  p.pre_desc = (int2*)w;
  p.rec_own = (int64_t)slot_rows();
  p.rec_pre = p.rec_own + (int64_t)p.B * p.Hq;
}

bool decode_mfma_supported(const DecodeParams& p, int q_dt, int kv_dt) {
  // bf16 or fp32 queries over bf16 or e4m3 caches; fp16 queries over fp16
  // or e4m3; fp32 queries over fp32; any over int8 (with block scales)
  if (kv_dt == kI8) {
    if (q_dt != kBF16 && q_dt != kF16 && q_dt != kF32) return false;
  } else if (q_dt == kBF16 || q_dt == kF32) {
    if (kv_dt != kBF16 && kv_dt != kE4M3 && (kv_dt != kF32 || q_dt != kF32)) return false;
  } else if (q_dt == kF16) {
    if (kv_dt != kF16 && kv_dt != kE4M3) return false;
  } else {
    return false;
  }
  if (p.bs != 16 || (p.D != 64 && p.D != 128)) return false;
  if (p.G != 1 && p.G != 2 && p.G != 4 && p.G != 8 && p.G != 16) return false;
  if (p.NB < 1) return false;  // invalid block ids are redirected to block 0 (then masked)
  // partial-row indices and descriptors are int32
  if ((uint64_t)total_rows(p.B, p.Hq) >= (uint64_t)INT32_MAX / 2) return false;
  const int kb = kv_dt == kE4M3 || kv_dt == kI8 ? 1 : (kv_dt == kF32 ? 4 : 2);
  // K: token rows with unit channel stride, 16-byte aligned (token stride D
  // in the native / paired layouts, any multiple of 16 bytes token-major).
  // V: the native tile [D][bs] (token stride 1, channel stride bs), or
  // token-major rows (channel stride 1) -- block/head strides free.
  if (p.k_s[3] != 1) return false;
  for (int i = 0; i < 3; ++i)
    if ((p.k_s[i] * kb) % 16 != 0) return false;
  const bool v_native = p.v_s[1] == 1 && p.v_s[3] == 16;
  const bool v_tok = p.v_s[3] == 1 && p.v_s[1] != 1 && (p.v_s[1] * kb) % 16 == 0;
  if (!v_native && !v_tok) return false;
  // native V rides with the native K tile (token stride D)
  if (v_native && p.k_s[1] != p.D) return false;
  if ((p.v_s[0] * kb) % 16 != 0 || (p.v_s[2] * kb) % 16 != 0) return false;
  if (v_native && (p.v_s[3] * kb) % 16 != 0) return false;
  if (!aligned16(p.k) || !aligned16(p.v)) return false;
  // q rows: 16-byte aligned slices; out rows: aligned groups of 4 (8 bytes
  // of 16-bit codes, 16 bytes of fp32).
  const int qb = q_dt == kF32 ? 4 : 2, oal = q_dt == kF32 ? 16 : 8;
  if (!aligned16(p.q) || (p.q_sb * qb) % 16 != 0 || (p.q_sh * qb) % 16 != 0) return false;
  if (((uintptr_t)p.out & (oal - 1)) != 0 || (p.o_sb * qb) % oal != 0 || (p.o_sh * qb) % oal != 0) return false;
  return true;
}

int32_t launch_decode_mfma(const DecodeParams& p, int q_dt, int kv_dt, hipStream_t stream) {
  return launch_any(p, q_dt, kv_dt, stream);
}

int32_t launch_decode_mfma(const DecodeWeightsParams& p, int q_dt, int kv_dt, hipStream_t stream) {
  return launch_any(p, q_dt, kv_dt, stream);
}

}  // namespace cf
