// Accounts of a decode step: what each cached token drew of the step's
// attention weight, added to what it drew before.
//
//   w[b, hw, t] = (t newest ? 0 : decay * w[b, hw, t]) + sum_h p[b, h, t],
//   p[b, h, t] = exp(s[b, h, t] - m[b, h]) / l[b, h],
// h over the query heads of account hw.  A row's l is known only once all its
// tokens have been seen, so the decode kernels leave their scores (4 bytes a
// head and token, against 2 * D * element bytes a KV head and token of K and
// V) and the final (m, l), and this kernel forms the weights: every account
// entry by one thread, no atomics.
//
// Bound by bytes: the scores, mostly still in the last-level cache, and the
// accounts read and written.
#include "cf_device.hpp"
#include "cf_host.hpp"
#include "decode_params.hpp"

namespace cf {

namespace {

constexpr int kTokens = 4;  // of a thread

template <bool LOG2>
__device__ __forceinline__ float weight_of(float s, float mref, float inv) {
  if (s == -INFINITY) return 0.0f;  // masked, or lost to a score of +inf
  return (LOG2 ? __builtin_amdgcn_exp2f(s - mref) : expf(s - mref)) * inv;
}

template <bool LOG2, bool VEC>
__global__ __launch_bounds__(256) void decode_weights_kernel(DecodeWeightsParams p) {
  const int chunks = (p.Mb * p.bs + 256 * kTokens - 1) / (256 * kTokens);
  const int bh = blockIdx.x / chunks, b = bh / p.Hw, hw = bh - b * p.Hw;
  const int t0 = ((blockIdx.x - bh * chunks) * 256 + threadIdx.x) * kTokens;
  const int ctx = p.seq_lens[(int64_t)b * p.sl_s], cap = p.Mb * p.bs, len = ctx < cap ? ctx : cap;
  if (t0 >= len) return;
  const int heads = p.Hq / p.Hw;
  const float* fin = p.ws_fin + ((int64_t)b * p.Hq + hw * heads) * 2;
  const int first = hw * heads;
  float acc[kTokens] = {0.0f, 0.0f, 0.0f, 0.0f};
  for (int h0 = 0; h0 < heads; h0 += p.G) {  // KV heads
    const float* s = p.ws_s + ((int64_t)b * p.Hq + first + h0) * p.s_cap + score_at(t0, 0, p.G);
#pragma unroll 4
    for (int g = 0; g < p.G; ++g) {
      const float m = fin[2 * (h0 + g)], l = fin[2 * (h0 + g) + 1];
      const float mref = m == -INFINITY ? 0.0f : m;
      const float inv = l == 0.0f ? 0.0f : 1.0f / l;  // (l NaN: so are the weights)
      const float4 v = *(const float4*)(s + g * 16);
      acc[0] += weight_of<LOG2>(v.x, mref, inv);
      acc[1] += weight_of<LOG2>(v.y, mref, inv);
      acc[2] += weight_of<LOG2>(v.z, mref, inv);
      acc[3] += weight_of<LOG2>(v.w, mref, inv);
    }
  }
  float* w = p.weights + (int64_t)b * p.w_sb + (int64_t)hw * p.w_sh + t0;
  const bool keep = p.decay != 0.0f;  // (0: what was there is not read)
  float old[kTokens] = {0.0f, 0.0f, 0.0f, 0.0f};
  if (VEC && t0 + kTokens <= len) {
    if (keep) {
      const float4 v = *(const float4*)w;
      old[0] = v.x;
      old[1] = v.y;
      old[2] = v.z;
      old[3] = v.w;
    }
#pragma unroll
    for (int i = 0; i < kTokens; ++i) acc[i] += t0 + i == ctx - 1 || !keep ? 0.0f : old[i] * p.decay;
    *(float4*)w = make_float4(acc[0], acc[1], acc[2], acc[3]);
    return;
  }
#pragma unroll
  for (int i = 0; i < kTokens; ++i)
    if (t0 + i < len) w[i] = acc[i] + (t0 + i == ctx - 1 || !keep ? 0.0f : w[i] * p.decay);
}

}  // namespace

int32_t launch_decode_weights(const DecodeWeightsParams& p, bool log2_units, hipStream_t stream) {
  const int64_t blocks = ceil_div((int64_t)p.Mb * p.bs, 256 * kTokens) * p.B * p.Hw;
  if (blocks == 0) return CF_OK;
  if (blocks >= (int64_t)INT32_MAX) {
    set_error("decode weights: too many accounts");
    return CF_ERR_UNSUPPORTED;
  }
  const bool vec = ((uintptr_t)p.weights & 15) == 0 && p.w_sb % 4 == 0 && p.w_sh % 4 == 0;
  const dim3 grid((unsigned)blocks);
  ProfileScope prof("cf_decode_weights", stream);
  if (log2_units) {
    if (vec) CF_LAUNCH((decode_weights_kernel<true, true>), grid, dim3(256), 0, stream, p);
    else CF_LAUNCH((decode_weights_kernel<true, false>), grid, dim3(256), 0, stream, p);
  } else {
    if (vec) CF_LAUNCH((decode_weights_kernel<false, true>), grid, dim3(256), 0, stream, p);
    else CF_LAUNCH((decode_weights_kernel<false, false>), grid, dim3(256), 0, stream, p);
  }
  CF_HIP_CHECK(hipGetLastError());
  return CF_OK;
}

}  // namespace cf
