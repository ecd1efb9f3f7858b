// Accounts of a decode step: what each cached token drew of the step's
// attention weight, added to what it drew before.
//
//   w[b, hw, t] = (t newest ? 0 : decay * w[b, hw, t]) + sum_h p[b, h, t],
//   p[b, h, t] = exp(s[b, h, t] - m[b, h]) / l[b, h],
// h over the query heads of account hw.  A row's l is known only once all its
// tokens have been seen, so the decode kernels leave their scores (4 bytes a
// head and token, against 2 * D * element bytes a KV head and token of K and
// V), and the weights are formed afterwards: every account entry by one thread,
// no atomics.  Few accounts of one KV head each are formed in the launch that
// joins the rows (account_block); this kernel forms the others, those of all
// heads, and those of calls whose rows need no joining.
//
// Bound by bytes: the scores, mostly still in the last-level cache, and the
// accounts read and written (64 sequences of 1,024 to 8,192 tokens, 32 / 8 heads:
// 38 MB of scores and 18 MB in 13.8 us).
#include "cf_device.hpp"
#include "cf_host.hpp"
#include "decode_account.hpp"
#include "decode_params.hpp"

namespace cf {

namespace {

template <bool LOG2>
__global__ __launch_bounds__(256) void decode_weights_kernel(DecodeWeightsParams p, bool vec) {
  const int chunks = (p.Mb * p.bs + kAccountBlock - 1) / kAccountBlock;
  const int bh = blockIdx.x / chunks, b = bh / p.Hw, hw = bh - b * p.Hw;
  const int t0 = ((blockIdx.x - bh * chunks) * 256 + threadIdx.x) * kAccountTokens;
  const int ctx = p.seq_lens[(int64_t)b * p.sl_s], cap = p.Mb * p.bs, len = ctx < cap ? ctx : cap;
  if (t0 >= len) return;
  const int heads = p.Hq / p.Hw, first = hw * heads;
  const float* fin = p.ws_fin + ((int64_t)b * p.Hq + first) * 2;
  float acc[kAccountTokens] = {0.0f, 0.0f, 0.0f, 0.0f};
  for (int h0 = 0; h0 < heads; h0 += p.G) {  // KV heads
    const float* s = p.ws_s + ((int64_t)b * p.Hq + first + h0) * p.s_cap + score_at(t0, 0, p.G);
#pragma unroll 4
    for (int g = 0; g < p.G; ++g) {
      const float2 f = finished(fin[2 * (h0 + g)], fin[2 * (h0 + g) + 1]);
      const float4 v = *(const float4*)(s + g * 16);
      acc[0] += weight_of<LOG2>(v.x, f.x, f.y);
      acc[1] += weight_of<LOG2>(v.y, f.x, f.y);
      acc[2] += weight_of<LOG2>(v.z, f.x, f.y);
      acc[3] += weight_of<LOG2>(v.w, f.x, f.y);
    }
  }
  AccountRow(p, b, hw, t0, len, ctx, vec).add(acc);
}

}  // namespace

int32_t launch_decode_weights(const DecodeWeightsParams& p, bool log2_units, hipStream_t stream) {
  const int64_t blocks = account_blocks(p);
  if (blocks == 0) return CF_OK;
  if (blocks >= (int64_t)INT32_MAX) {
    set_error("decode weights: too many accounts");
    return CF_ERR_UNSUPPORTED;
  }
  const dim3 grid((unsigned)blocks);
  ProfileScope prof("cf_decode_weights", stream);
  if (log2_units) CF_LAUNCH((decode_weights_kernel<true>), grid, dim3(256), 0, stream, p, accounts_aligned(p));
  else CF_LAUNCH((decode_weights_kernel<false>), grid, dim3(256), 0, stream, p, accounts_aligned(p));
  CF_HIP_CHECK(hipGetLastError());
  return CF_OK;
}

}  // namespace cf
