// Eviction from a paged KV cache by accumulated attention weight.
//
// evict_select: of a sequence's len cached tokens every head keeps
// n = min(len, budget): first the protected ones (position < sink, or
// position >= seen - recent), then those of the greatest accumulated weight,
// NaN above all numbers as in a descending sort, equal weights by the lower
// index.  Attention does not ask in which order a sequence's tokens lie in
// its slots (their rows hold their positions), so a kept token with an index
// below n stays where it is, and the k-th kept token at or above n (a mover)
// takes the k-th slot below n whose token is not kept (a hole):
//   keep[j] = the index whose token belongs in slot j, -1 for j >= n.
// No mover's slot is ever a hole, so the moves are independent of each other,
// and a step that evicts one token a head moves one row a head instead of
// closing up the whole cache.
//
// evict_move: K and V rows, weights and positions of every slot with
// keep[j] != j, from keep[j].
#include "cf_device.hpp"
#include "cf_host.hpp"
#include "kv_evict.hpp"

namespace cf {

namespace {

// ---- select ------------------------------------------------------------------
//
// One workgroup a (sequence, head).  A weight becomes a 32-bit key in the
// order above (protected tokens the greatest key, indices past the sequence
// 0), held in registers: wave v's item e of lane l is index
// (v * E + e) * 64 + l, so loads are whole runs and ranks follow the index.
// The budget-th greatest key is found from the top bit downwards, a count of
// the keys at or above a candidate for each bit; a count is one comparison a
// key and scalar popcounts, where a histogram's LDS atomics would meet in few
// bins (accounts differ by little in their leading bits).

__device__ __forceinline__ uint32_t key_of(float w) {
  if (w != w) return 0xFFFFFFFEu;
  const uint32_t u = f2u(w + 0.0f);  // -0 and +0 are equal
  return (u >> 31) ? ~u : u | 0x80000000u;
}

constexpr uint32_t kSafe = 0xFFFFFFFFu;  // a protected token's key

struct SelectRow {
  const float* w;
  const int32_t* pos;  // null: a slot's index is its position
  int len, kept, first, sink;
  int64_t recent_from;  // positions at or above it are protected
  __device__ __forceinline__ uint32_t key(int i) const {
    if (i >= len) return 0u;
    const uint32_t k = key_of(w[i]);
    const int64_t at = pos == nullptr ? i : (i < kept ? (int64_t)pos[i] : (int64_t)first + i);
    return at < sink || at >= recent_from ? kSafe : k;
  }
};

// Lanes below this one whose bit is set.
__device__ __forceinline__ int rank_in(uint64_t mask) {
  return __builtin_amdgcn_mbcnt_hi((uint32_t)(mask >> 32), __builtin_amdgcn_mbcnt_lo((uint32_t)mask, 0u));
}

// Sum of v over the waves before this one, and over all (v wave-uniform).
// `slot`: LDS of one int a wave that no wave still reads.
template <int WAVES>
__device__ __forceinline__ int2 before_and_all(int* slot, int v, int wave) {
  if ((threadIdx.x & 63) == 0) slot[wave] = v;
  __syncthreads();
  int before = 0, all = 0;
#pragma unroll
  for (int i = 0; i < WAVES; ++i) {
    const int x = slot[i];
    all += x;
    before += i < wave ? x : 0;
  }
  return make_int2(before, all);
}

constexpr int kListCap = 4096;  // movers handed to their holes at a time

// E > 0: up to E * THREADS keys in registers; E == 0: any number, read again
// for every use.
template <int THREADS, int E>
__global__ __launch_bounds__(THREADS) void evict_select_kernel(EvictSelectParams p) {
  constexpr int WAVES = THREADS / 64;
  __shared__ int counts[4][WAVES];
  __shared__ int list[kListCap];
  const int b = blockIdx.x / p.H, h = blockIdx.x - b * p.H;
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int raw = p.lens[(int64_t)b * p.l_s];
  const int len = raw < 0 ? 0 : (raw < p.S ? raw : p.S);
  const int budget = p.budget;
  int32_t* keep = p.keep + (int64_t)b * p.k_sb + (int64_t)h * p.k_sh;
  if (h == 0 && threadIdx.x == 0) p.new_lens[(int64_t)b * p.n_s] = len < budget ? len : budget;
  if (len <= budget) {
    for (int j = threadIdx.x; j < budget; j += THREADS) keep[j] = j < len ? j : -1;
    return;
  }
  SelectRow row;
  row.w = p.weights + (int64_t)b * p.w_sb + (int64_t)h * p.w_sh;
  row.pos = p.positions == nullptr ? nullptr : p.positions + (int64_t)b * p.p_sb + (int64_t)h * p.p_sh;
  row.len = len;
  row.sink = p.sink;
  const int seen = p.positions == nullptr ? len : p.seen[(int64_t)b * p.seen_s];
  row.kept = p.positions == nullptr ? 0 : p.kept[(int64_t)b * p.kept_s];
  row.first = seen - len;
  row.recent_from = (int64_t)seen - p.recent;

  const int items = E > 0 ? E : (len + THREADS - 1) / THREADS;  // of a lane
  const int base = wave * items * 64 + lane;
  uint32_t reg[E > 0 ? E : 1];
  if constexpr (E > 0) {
#pragma unroll
    for (int e = 0; e < E; ++e) reg[e] = row.key(base + e * 64);
  }
  auto each = [&](auto f) {
    if constexpr (E > 0) {
#pragma unroll
      for (int e = 0; e < E; ++e) f(base + e * 64, reg[e]);
    } else {
      for (int e = 0; e < items; ++e) f(base + e * 64, row.key(base + e * 64));
    }
  };

  // the greatest key that at least `budget` keys reach
  uint32_t top = 0u;
  for (int bit = 31; bit >= 0; --bit) {
    const uint32_t cand = top | (1u << bit);
    int n = 0;
    each([&](int, uint32_t k) { n += __popcll(__ballot(k >= cand)); });
    if (before_and_all<WAVES>(counts[bit & 1], n, wave).y >= budget) top = cand;
  }
  // of the keys equal to it, the lowest indices are kept
  int above = 0, equal = 0;
  each([&](int, uint32_t k) {
    above += __popcll(__ballot(k > top));
    equal += __popcll(__ballot(k == top));
  });
  const int all_above = before_and_all<WAVES>(counts[2], above, wave).y;
  const int eq0 = before_and_all<WAVES>(counts[3], equal, wave).x;
  const int want = budget - all_above;
  // holes and movers of the waves before this one
  int eq = eq0, holes = 0, movers = 0;
  each([&](int i, uint32_t k) {
    const uint64_t em = __ballot(k == top);
    const bool kept = k > top || (k == top && eq + rank_in(em) < want);
    eq += __popcll(em);
    holes += __popcll(__ballot(i < budget && !kept));
    movers += __popcll(__ballot(i >= budget && kept));
  });
  const int hole0 = before_and_all<WAVES>(counts[0], holes, wave).x;
  const int2 mv = before_and_all<WAVES>(counts[1], movers, wave);
  // movers and holes meet in LDS, kListCap at a time
  for (int at = 0; at == 0 || at < mv.y; at += kListCap) {
    int r = mv.x;
    eq = eq0;
    each([&](int i, uint32_t k) {
      const uint64_t em = __ballot(k == top);
      const bool kept = k > top || (k == top && eq + rank_in(em) < want);
      eq += __popcll(em);
      const uint64_t mm = __ballot(i >= budget && kept);
      const int mine = r + rank_in(mm) - at;
      if (i >= budget && kept && mine >= 0 && mine < kListCap) list[mine] = i;
      r += __popcll(mm);
    });
    __syncthreads();
    r = hole0;
    eq = eq0;
    each([&](int i, uint32_t k) {
      const uint64_t em = __ballot(k == top);
      const bool kept = k > top || (k == top && eq + rank_in(em) < want);
      eq += __popcll(em);
      const uint64_t hm = __ballot(i < budget && !kept);
      const int mine = r + rank_in(hm) - at;
      if (i < budget) {
        if (kept) {
          if (at == 0) keep[i] = i;
        } else if (mine >= 0 && mine < kListCap) {
          keep[i] = list[mine];
        }
      }
      r += __popcll(hm);
    });
    __syncthreads();
  }
}

// ---- move --------------------------------------------------------------------
//
// A workgroup takes kMoveSlots slots of one (sequence, account head): it
// lists those whose token comes from elsewhere, moves their weights and
// positions, and copies the listed rows of every KV head of the account
// (one, or all of them).

constexpr int kMoveSlots = 256;

template <class T>
__device__ __forceinline__ void copy_rows(const EvictMoveParams& p, int which, int h0, int nh, const int2* from_to,
                                          int n) {
  T* base = (T*)p.cache[which];
  const int64_t* s = p.c_s[which];
  const int per = nh * p.D;
  for (int u = threadIdx.x; u < n * per; u += 256) {
    const int k = u / per, r = u - k * per;
    const int h = h0 + r / p.D, d = r % p.D;
    const int2 m = from_to[k];
    const int64_t src = (int64_t)(m.x / p.bs) * s[0] + (int64_t)(m.x % p.bs) * s[1];
    const int64_t dst = (int64_t)(m.y / p.bs) * s[0] + (int64_t)(m.y % p.bs) * s[1];
    const int64_t at = (int64_t)h * s[2] + (int64_t)d * s[3];
    base[dst + at] = base[src + at];
  }
}

template <class T>
__global__ __launch_bounds__(256) void evict_move_kernel(EvictMoveParams p) {
  __shared__ int2 list[kMoveSlots];  // (source, destination) as block * bs + offset
  __shared__ int count;
  const int chunks = (p.budget + kMoveSlots - 1) / kMoveSlots;
  const int bh = blockIdx.x / chunks, b = bh / p.Hw, h = bh - b * p.Hw;
  const int j = (blockIdx.x - bh * chunks) * kMoveSlots + threadIdx.x;
  if (threadIdx.x == 0) count = 0;
  __syncthreads();
  const int raw = p.lens[(int64_t)b * p.l_s];
  const int src = j < p.budget ? p.keep[(int64_t)b * p.k_sb + (int64_t)h * p.k_sh + j] : -1;
  // (a source outside the tables cannot come from a selection)
  const int cap = p.Mb * p.bs;
  if (src >= 0 && src < cap && src < p.S && j < cap && j < p.S) {
    if (p.positions != nullptr) {
      const int kept = p.kept[(int64_t)b * p.kept_s];
      if (src != j || j >= kept) {
        const int len = raw < 0 ? 0 : (raw < p.S ? raw : p.S);
        int32_t* pos = p.positions + (int64_t)b * p.p_sb + (int64_t)h * p.p_sh;
        pos[j] = src < kept ? pos[src] : p.seen[(int64_t)b * p.seen_s] - len + src;
      }
    }
    if (src != j) {
      if (p.weights != nullptr) {
        float* w = p.weights + (int64_t)b * p.w_sb + (int64_t)h * p.w_sh;
        w[j] = w[src];
      }
      const int32_t* t = p.tables + (int64_t)b * p.t_sb;
      const int from = t[(int64_t)(src / p.bs) * p.t_sm], to = t[(int64_t)(j / p.bs) * p.t_sm];
      if (from >= 0 && from < p.NB && to >= 0 && to < p.NB) {
        const int at = atomicAdd(&count, 1);  // (the order of independent copies)
        list[at] = make_int2(from * p.bs + src % p.bs, to * p.bs + j % p.bs);
      }
    }
  }
  __syncthreads();
  const int n = count;
  if (n == 0) return;
  const int nh = p.Hw == 1 ? p.Hkv : 1, h0 = p.Hw == 1 ? 0 : h;
  copy_rows<T>(p, 0, h0, nh, list, n);
  copy_rows<T>(p, 1, h0, nh, list, n);
}

template <int THREADS, int E>
int32_t launch_select_t(const EvictSelectParams& p, hipStream_t stream) {
  ProfileScope prof("cf_evict_select", stream);
  CF_LAUNCH((evict_select_kernel<THREADS, E>), dim3((unsigned)(p.H * p.B)), dim3(THREADS), 0, stream, p);
  CF_HIP_CHECK(hipGetLastError());
  return CF_OK;
}

}  // namespace

int32_t launch_evict_select(const EvictSelectParams& p, hipStream_t stream) {
  if (p.S <= 256 * 4) return launch_select_t<256, 4>(p, stream);
  if (p.S <= 256 * 16) return launch_select_t<256, 16>(p, stream);
  if (p.S <= 1024 * 16) return launch_select_t<1024, 16>(p, stream);
  if (p.S <= 1024 * 32) return launch_select_t<1024, 32>(p, stream);
  return launch_select_t<1024, 0>(p, stream);
}

int32_t launch_evict_move(const EvictMoveParams& p, int elem_bytes, hipStream_t stream) {
  const dim3 grid((unsigned)(ceil_div(p.budget, kMoveSlots) * p.Hw * p.B));
  ProfileScope prof("cf_evict_move", stream);
  switch (elem_bytes) {
    case 1: CF_LAUNCH((evict_move_kernel<uint8_t>), grid, dim3(256), 0, stream, p); break;
    case 2: CF_LAUNCH((evict_move_kernel<uint16_t>), grid, dim3(256), 0, stream, p); break;
    default: CF_LAUNCH((evict_move_kernel<uint32_t>), grid, dim3(256), 0, stream, p); break;
  }
  CF_HIP_CHECK(hipGetLastError());
  return CF_OK;
}

}  // namespace cf
