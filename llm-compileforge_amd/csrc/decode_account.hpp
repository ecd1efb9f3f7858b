// The accounts of a decode step: what each cached token drew of the step's
// attention weight, added to what it drew before (device code).
#pragma once

#include "cf_device.hpp"
#include "decode_params.hpp"

namespace cf {

constexpr int kAccountTokens = 4;                      // of a thread
constexpr int kAccountBlock = 256 * kAccountTokens;  // of a workgroup

// A score's weight; mref, inv: the row's reference and 1 / sum.
template <bool LOG2>
__device__ __forceinline__ float weight_of(float s, float mref, float inv) {
  if (s == -INFINITY) return 0.0f;  // masked, or lost to a score of +inf
  return (LOG2 ? __builtin_amdgcn_exp2f(s - mref) : expf(s - mref)) * inv;
}

// (reference, 1 / sum) of a row from its final (m, l) (l NaN: so are the weights).
__device__ __forceinline__ float2 finished(float m, float l) {
  return make_float2(m == -INFINITY ? 0.0f : m, l == 0.0f ? 0.0f : 1.0f / l);
}

// Tokens t0 .. + 3 of an account of len tokens, whose newest is ctx - 1: the sums
// and what the account held of them.  vec: the row is 16-byte aligned.
struct AccountRow {
  float* w;
  int t0, len, ctx;
  float decay;
  bool vec;
  float4 old;

  __device__ __forceinline__ AccountRow(const DecodeWeightsParams& p, int b, int hw, int first, int length, int context,
                                        bool aligned)
      : w(p.weights + (int64_t)b * p.w_sb + (int64_t)hw * p.w_sh + first), t0(first), len(length), ctx(context),
        decay(p.decay), vec(aligned && first + kAccountTokens <= length), old(make_float4(0.0f, 0.0f, 0.0f, 0.0f)) {
    if (vec && decay != 0.0f) old = *(const float4*)w;  // (0: what was there is not read)
  }
  __device__ __forceinline__ void add(const float* acc) const {
    const bool keep = decay != 0.0f;
    if (vec) {
      const float was[kAccountTokens] = {old.x, old.y, old.z, old.w};
      float v[kAccountTokens];
#pragma unroll
      for (int i = 0; i < kAccountTokens; ++i) v[i] = acc[i] + (t0 + i == ctx - 1 || !keep ? 0.0f : was[i] * decay);
      *(float4*)w = make_float4(v[0], v[1], v[2], v[3]);
      return;
    }
#pragma unroll
    for (int i = 0; i < kAccountTokens; ++i)
      if (t0 + i < len) w[i] = acc[i] + (t0 + i == ctx - 1 || !keep ? 0.0f : w[i] * decay);
  }
};

// kAccountBlock tokens of one KV head's account (block `block` of the call's),
// next to the kernel that joins the rows: the (m, l) of the head's rows are formed
// from the decode kernel's partials here, too, while the scores are on their way.
// `parts` gives them: count (0: the row's (m, l) are in ws_fin) and ml(g, k).
// fin: G pairs of LDS.
template <bool LOG2, class Parts>
__device__ __forceinline__ void account_block(const DecodeWeightsParams& p, int block, float2* fin, bool vec) {
  typedef float Four __attribute__((ext_vector_type(4)));
  constexpr int kHold = 8;  // heads whose scores are in flight at a time
  const int chunks = (p.Mb * p.bs + kAccountBlock - 1) / kAccountBlock;
  const int bh = block / chunks, b = bh / p.Hkv, h = bh - b * p.Hkv, base = (block - bh * chunks) * kAccountBlock;
  const int ctx = p.seq_lens[(int64_t)b * p.sl_s], cap = p.Mb * p.bs, len = ctx < cap ? ctx : cap;
  if (base >= len) return;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
  const int t0 = base + (int)threadIdx.x * kAccountTokens;
  const int64_t row0 = (int64_t)b * p.Hq + h * p.G;
  // (threads past the end read the last tokens' scores)
  const float* s = p.ws_s + row0 * p.s_cap + score_at(min(t0, (len - 1) & ~3), 0, p.G);
  Four v[kHold];
#pragma unroll
  for (int i = 0; i < kHold; ++i) v[i] = *(const Four*)(s + min(i, p.G - 1) * 16);
  const AccountRow row(p, b, h, t0, len, ctx, vec);
  const Parts parts(p, b, h);
  for (int g = wave; g < p.G; g += 4) {
    float M = -INFINITY, L = 0.0f;
    if (parts.count == 0) {
      M = p.ws_fin[(row0 + g) * 2];
      L = p.ws_fin[(row0 + g) * 2 + 1];
    }
    for (int k0 = 0; k0 < parts.count; k0 += 64) {
      const bool live = k0 + lane < parts.count;
      const float2 ml = live ? parts.ml(g, k0 + lane) : make_float2(-INFINITY, 0.0f);
      const float mn = fmaxf(M, wave_max(ml.x));
      auto scale = [&](float m) { return m == -INFINITY ? 1.0f : (LOG2 ? __builtin_amdgcn_exp2f(m - mn) : expf(m - mn)); };
      L = L * scale(M) + wave_sum(live ? ml.y * scale(ml.x) : 0.0f);
      M = mn;
    }
    if (lane == 0) fin[g] = finished(M, L);
  }
  __syncthreads();
  if (t0 >= len) return;
  float acc[kAccountTokens] = {0.0f, 0.0f, 0.0f, 0.0f};
  for (int g0 = 0; g0 < p.G; g0 += kHold) {
    if (g0 > 0) {
#pragma unroll
      for (int i = 0; i < kHold; ++i) v[i] = *(const Four*)(s + min(g0 + i, p.G - 1) * 16);
    }
#pragma unroll
    for (int i = 0; i < kHold; ++i) {
      if (g0 + i < p.G) {
        const float2 f = fin[g0 + i];
#pragma unroll
        for (int t = 0; t < kAccountTokens; ++t) acc[t] += weight_of<LOG2>(v[i][t], f.x, f.y);
      }
    }
  }
  row.add(acc);
}

}  // namespace cf
