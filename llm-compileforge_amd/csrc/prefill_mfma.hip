// The chunked-prefill kernels (prefill_item.hpp) of caches with a scale for each KV head, or none: launchers, their
// workspace and what they take.
#include "prefill_item.hpp"

namespace cf {

namespace {

uint64_t pad256(uint64_t x) { return (x + 255) & ~(uint64_t)255; }

}  // namespace

bool prefill_supported(const PrefillParams& p, int q_dt, int kv_dt) {
  // bf16 queries over bf16 or e4m3 caches; fp16 queries over fp16 or e4m3;
  // either over int8 (with block scales)
  if (kv_dt == kI8) {
    if (q_dt != kBF16 && q_dt != kF16) return false;
  } else if (q_dt == kBF16) {
    if (kv_dt != kBF16 && kv_dt != kE4M3) return false;
  } else if (q_dt == kF16) {
    if (kv_dt != kF16 && kv_dt != kE4M3) return false;
  } else {
    return false;
  }
  if (p.D != 64 && p.D != 128) return false;
  if (p.G != 1 && p.G != 2 && p.G != 4 && p.G != 8 && p.G != 16) return false;
  if (p.NB < 1) return false;
  const int kb = kv_dt == kE4M3 || kv_dt == kI8 ? 1 : 2;
  // native (K token rows of head_dim, V channel rows of 16 tokens) or
  // token-major (the reference's layout: both caches in token rows)
  const bool native = p.k_s[3] == 1 && p.k_s[1] == p.D && p.v_s[1] == 1 && p.v_s[3] == 16;
  const bool token_major = p.k_s[3] == 1 && p.v_s[3] == 1 && p.v_s[1] != 1 && (p.k_s[1] * kb) % 16 == 0 &&
                           (p.v_s[1] * kb) % 16 == 0;
  if (!native && !token_major) return false;
  // in-block offsets (15 token rows plus a row) are 32-bit in the kernel
  const int64_t max_off = 16 * (p.k_s[1] > p.v_s[1] ? p.k_s[1] : p.v_s[1]) * kb + (int64_t)p.D * 16 * kb;
  if (p.k_s[1] < 0 || p.v_s[1] < 0 || max_off >= ((int64_t)1 << 32)) return false;
  if ((p.k_s[0] * kb) % 16 || (p.k_s[2] * kb) % 16 || (p.v_s[0] * kb) % 16 || (p.v_s[2] * kb) % 16) return false;
  if (((uintptr_t)p.k & 15) || ((uintptr_t)p.v & 15)) return false;
  if (((uintptr_t)p.q & 15) || (p.q_sr * 2) % 16 || (p.q_sh * 2) % 16) return false;
  if (((uintptr_t)p.out & 7) || (p.o_sr * 2) % 8 || (p.o_sh * 2) % 8) return false;
  return true;
}

int prefill_rows_per_item(int G) { return kCols / G; }

// Slots for the pieces of a direct launch, one per resident workgroup; none
// when the call may hold more items than that (queued launches cut nothing).
int64_t split_slots_of(int64_t max_items, int64_t D) {
  const int64_t w = std::min<int64_t>((int64_t)prefill_cus() * item_blocks_per_cu(D, true), kDirectItems);
  return max_items <= w ? w : 0;
}

// Workspace: [chunks int4 x N][items int4 x max_items][header 12 int], and
// for direct launches that cut items [merge records 2 int4 x max_items][(m, l)
// float2 x 128 per slot][o float x 128 x D per slot].  A workspace that ends
// with the header serves every call: it is then queued.
uint64_t queue_workspace_bytes(int64_t N, int64_t max_items) {
  return pad256((uint64_t)N * 16) + pad256((uint64_t)max_items * 16) + 256;
}

uint64_t slot_workspace_bytes(int64_t max_items, int64_t D, uint64_t slots) {
  if (slots == 0) return 0;
  return pad256((uint64_t)max_items * 32) + pad256(slots * kCols * 8) + slots * kCols * (uint64_t)D * 4;
}

uint64_t prefill_workspace_bytes(int64_t Tq, int64_t N, int64_t Hq, int64_t Hkv, int64_t D) {
  const int64_t G = Hkv > 0 ? Hq / Hkv : 1;
  const int64_t RB = std::max<int64_t>(G > 0 ? kCols / G : 1, 1);
  const int64_t max_items = (Tq / RB + N) * Hkv;
  return queue_workspace_bytes(N, max_items) +
         slot_workspace_bytes(max_items, D, (uint64_t)split_slots_of(max_items, D));
}

uint64_t prefill_bind_workspace(PrefillParams& p, void* workspace, uint64_t bytes) {
  const uint64_t base = queue_workspace_bytes(p.N, p.max_items);
  if (bytes < base) return base;
  uint64_t slots = (uint64_t)split_slots_of(p.max_items, p.D);
  if (bytes - base < slot_workspace_bytes(p.max_items, p.D, slots)) slots = 0;
  p.split_slots = (int)slots;
  char* w = (char*)workspace;
  p.chunks = (int4*)w;
  w += pad256((uint64_t)p.N * 16);
  p.items = (int4*)w;
  w += pad256((uint64_t)p.max_items * 16);
  p.header = (int*)w;
  p.splits = nullptr;
  p.ws_ml = nullptr;
  p.ws_o = nullptr;
  if (slots > 0) {
    w += 256;
    p.splits = (int4*)w;
    w += pad256((uint64_t)p.max_items * 32);
    p.ws_ml = (float2*)w;
    w += pad256(slots * kCols * 8);
    p.ws_o = (float4*)w;
  }
  return 0;
}

int32_t launch_prefill(PrefillParams& p, int q_dt, int kv_dt, hipStream_t stream) {
  if (q_dt == kF16) return kv_dt == kE4M3 ? launch_d<kF16, kE4M3>(p, stream) : launch_d<kF16, kF16>(p, stream);
  return kv_dt == kE4M3 ? launch_d<kBF16, kE4M3>(p, stream) : launch_d<kBF16, kBF16>(p, stream);
}

}  // namespace cf
