// The chunked-prefill kernels (prefill_item.hpp) of e4m3 caches with a scale for each block and head.
#include "prefill_item.hpp"

namespace cf {

int32_t launch_prefill_e4m3(PrefillBlockParams& p, int q_dt, hipStream_t stream) {
  return q_dt == kF16 ? launch_d<kF16, kE4M3>(p, stream) : launch_d<kBF16, kE4M3>(p, stream);
}

}  // namespace cf
