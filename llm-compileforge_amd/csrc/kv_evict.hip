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
#include "mfma_tile.hpp"

namespace cf {

namespace {

// ---- select ------------------------------------------------------------------
//
// One workgroup a (sequence, head).  A weight becomes a 32-bit key in the
// order above (protected tokens the greatest key, indices past the sequence
// 0), held in registers: wave v's item e of lane l is index
// (v * items + e) * 64 + l, so loads are whole runs and ranks follow the index.
// The budget-th greatest key is found in two steps: a histogram of the ten
// bits below the first in which keys differ (so that accounts, which share
// their leading bits, spread over its bins), and, among the keys of the bin
// that it lies in, a search two bits at a time by counts of the keys at or
// above the three candidates.  The bin's keys are gathered in LDS, a key a
// lane of one wave; if they are too many, a histogram of the bin's next ten
// bits comes first.  A workgroup is bound by its instructions a key (some 80)
// and the latency of its barriers and LDS steps.
// 64 sequences of 8 heads and 2,064 slots: 12.4 us, 13.6 with positions (8.4 and
// 12.6 MB); four of 30,000: 29.0 and 31.4.  What lies past a sequence's end in its
// buffer costs its loads: 2,064 tokens in 32,000 slots take 52 us.

__device__ __forceinline__ uint32_t key_of(float w) {
  if (w != w) return 0xFFFFFFFEu;
  const uint32_t u = f2u(w + 0.0f);  // -0 and +0 are equal
  return (u >> 31) ? ~u : u | 0x80000000u;
}

constexpr uint32_t kSafe = 0xFFFFFFFFu;  // a protected token's key

struct SelectRow {
  const float* w;
  const int32_t* pos;  // null: a slot's index is its position
  int last;             // of the buffer's slots
  int len, kept, first, sink;
  int64_t recent_from;  // positions at or above it are protected
  // (loads of indices past the end take the last one: they need no branch, so
  // all of a lane's are in flight together)
  __device__ __forceinline__ float weight(int i) const { return w[(uint32_t)min(i, last)]; }
  __device__ __forceinline__ int position(int i) const { return pos[(uint32_t)min(i, last)]; }
  __device__ __forceinline__ uint32_t key(int i, float wi, int stored) const {
    const int64_t at = pos != nullptr && i < kept ? (int64_t)stored : (int64_t)first + i;
    const uint32_t k = at < sink || at >= recent_from ? kSafe : key_of(wi);
    return i < len ? k : 0u;
  }
};

// Lanes below this one whose bit is set.
__device__ __forceinline__ int rank_in(uint64_t mask) {
  return __builtin_amdgcn_mbcnt_hi((uint32_t)(mask >> 32), __builtin_amdgcn_mbcnt_lo((uint32_t)mask, 0u));
}

// Sum over N consecutive lanes, N a power of two up to 16, of values that
// repeat every N lanes (rotations within a row of 16).
template <int N>
__device__ __forceinline__ int ring_sum(int v) {
  if constexpr (N > 8) v += __builtin_amdgcn_update_dpp(0, v, 0x128, 0xF, 0xF, false);
  if constexpr (N > 4) v += __builtin_amdgcn_update_dpp(0, v, 0x124, 0xF, 0xF, false);
  if constexpr (N > 2) v += __builtin_amdgcn_update_dpp(0, v, 0x122, 0xF, 0xF, false);
  if constexpr (N > 1) v += __builtin_amdgcn_update_dpp(0, v, 0x121, 0xF, 0xF, false);
  return __builtin_amdgcn_readfirstlane(v);
}

// The waves' values meet in LDS: each wave writes its own and reads all, a
// wave's a lane (one read, where a broadcast read of each would be 16).
// `slot`: LDS of a value a wave that no wave still reads.

// Sum of v over the waves before this one, and over all (v wave-uniform).
template <int WAVES>
__device__ __forceinline__ int2 before_and_all(int* slot, int v, int wave) {
  const int lane = threadIdx.x & 63;
  if (lane == 0) slot[wave] = v;
  __syncthreads();
  const int x = slot[lane & (WAVES - 1)];
  return make_int2(ring_sum<WAVES>((lane & (WAVES - 1)) < wave ? x : 0), ring_sum<WAVES>(x));
}

// a + b, at most 2^32 - 1 (a key that no unprotected token has).
__device__ __forceinline__ uint32_t plus(uint32_t a, uint32_t b) { return a > 0xFFFFFFFFu - b ? 0xFFFFFFFFu : a + b; }

constexpr int kListCap = 4096;  // movers handed to their holes at a time
constexpr int kBinBits = 10;    // of the histogram
constexpr int kLaneBins = (1 << kBinBits) / 64;
constexpr int kGather = 512;    // keys of one bin that are searched apart

// E > 0: up to E * THREADS keys in registers; E == 0: any number, read again
// for every use.
template <int THREADS, int E>
__global__ __launch_bounds__(THREADS) void evict_select_kernel(EvictSelectParams p) {
  constexpr int WAVES = THREADS / 64;
  __shared__ int counts[3][WAVES];
  __shared__ int4 votes[2][WAVES];
  __shared__ __align__(16) int hist[1 << kBinBits];
  __shared__ int found[3], gathered;
  __shared__ uint32_t few[kGather];
  const int b = blockIdx.x / p.H, h = blockIdx.x - b * p.H;
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int budget = p.budget;
  int32_t* keep = p.keep + (int64_t)b * p.k_sb + (int64_t)h * p.k_sh;
  SelectRow row;
  row.w = p.weights + (int64_t)b * p.w_sb + (int64_t)h * p.w_sh;
  row.pos = p.positions == nullptr ? nullptr : p.positions + (int64_t)b * p.p_sb + (int64_t)h * p.p_sh;
  row.last = p.S - 1;
  const int items = (p.S + THREADS - 1) / THREADS;  // of a lane
  const int base = wave * items * 64 + lane;
  // all loads go out before the length is known (the buffer is S long)
  uint32_t reg[E > 0 ? E : 1];
  if constexpr (E > 0) {
#pragma unroll
    for (int e = 0; e < E; ++e) reg[e] = p.S > 0 ? f2u(row.weight(base + e * 64)) : 0u;
  }
  const int raw = p.lens[(int64_t)b * p.l_s];
  const int seen = p.positions == nullptr ? 0 : p.seen[(int64_t)b * p.seen_s];
  row.kept = p.positions == nullptr ? 0 : p.kept[(int64_t)b * p.kept_s];
  const int len = raw < 0 ? 0 : (raw < p.S ? raw : p.S);
  if (h == 0 && threadIdx.x == 0) p.new_lens[(int64_t)b * p.n_s] = len < budget ? len : budget;
  if (len <= budget) {
    for (int j = threadIdx.x; j < budget; j += THREADS) keep[j] = j < len ? j : -1;
    return;
  }
  row.len = len;
  row.sink = p.sink;
  row.first = p.positions == nullptr ? 0 : seen - len;
  row.recent_from = (int64_t)row.first + len - p.recent;
  if constexpr (E > 0) {
    constexpr int kBatch = 8 < E ? 8 : E;  // positions in flight at a time
#pragma unroll
    for (int e0 = 0; e0 < E; e0 += kBatch) {
      int at[kBatch];
#pragma unroll
      for (int e = 0; e < kBatch; ++e) at[e] = row.pos != nullptr ? row.position(base + (e0 + e) * 64) : 0;
#pragma unroll
      for (int e = 0; e < kBatch; ++e) reg[e0 + e] = row.key(base + (e0 + e) * 64, u2f(reg[e0 + e]), at[e]);
    }
  }
  auto each = [&](auto f) {
    if constexpr (E > 0) {
#pragma unroll
      for (int e = 0; e < E; ++e) {
        if (e < items) f(base + e * 64, reg[e]);
      }
    } else {
      for (int e = 0; e < items; ++e) {
        const int i = base + e * 64;
        f(i, row.key(i, row.weight(i), row.pos != nullptr ? row.position(i) : 0));
      }
    }
  };

  // the range of the unprotected keys, and how many are protected (0 and kSafe
  // step aside: one below 0 and one above kSafe wrap round; the steps are taken
  // back once, after the workgroup's least and greatest are known, since lanes and
  // waves of nothing but 0 or kSafe hold the wrapped values until then)
  uint32_t lo = 0xFFFFFFFFu, hi = 0u;
  int safe = 0;
  each([&](int, uint32_t k) {
    lo = min(lo, k - 1u);
    hi = max(hi, k + 1u);
    safe += k == kSafe ? 1 : 0;
  });
  safe = wave_last(wave_incl_scan(safe, lane));
  lo = ~wave_umax(~lo);
  hi = wave_umax(hi);
  if (lane == 0) votes[0][wave] = make_int4((int)lo, (int)hi, safe, 0);
  __syncthreads();
  {
    const int4 v = votes[0][lane & (WAVES - 1)];
    lo = ~wave_umax(~(uint32_t)v.x) + 1u;
    hi = wave_umax((uint32_t)v.y) - 1u;
    safe = ring_sum<WAVES>(v.z);
  }
  // the greatest key that at least `budget` keys reach, how many keys are
  // above it and how many equal it
  uint32_t top = kSafe;
  int above = 0, equal = safe;
  if (safe < budget) {
    int first = lo == hi ? 0 : 32 - __builtin_clz(lo ^ hi);  // bits in which the keys left differ
    top = first == 32 ? 0u : hi >> first << first;           // the lowest that they can be
    above = safe;
    int members, shift;
    do {
      shift = first > kBinBits ? first - kBinBits : 0;
      for (int i = threadIdx.x; i < 1 << kBinBits; i += THREADS) hist[i] = 0;
      if (threadIdx.x == 0) gathered = 0;
      __syncthreads();
      each([&](int, uint32_t k) {
        const uint32_t at = (k - top) >> shift;
        if (at < 1u << (first - shift) && k - 1u < kSafe - 1u) atomicAdd(&hist[at], 1);  // (neither 0 nor protected)
      });
      __syncthreads();
      if (wave == 0) {  // lane l: kLaneBins bins, lane 0 the highest
        const int low = (63 - lane) * kLaneBins;
        int own[kLaneBins], sum = 0;
#pragma unroll
        for (int i = 0; i < kLaneBins; i += 4) {
          const int4 v = *(const int4*)&hist[low + i];
          own[i] = v.x, own[i + 1] = v.y, own[i + 2] = v.z, own[i + 3] = v.w;
          sum += (v.x + v.y) + (v.z + v.w);
        }
        int run = above + wave_incl_scan(sum, lane) - sum;
        if (run < budget && run + sum >= budget) {
#pragma unroll
          for (int i = kLaneBins - 1; i >= 0; --i) {
            if (run < budget && run + own[i] >= budget) {
              found[0] = low + i;
              found[1] = run;
              found[2] = own[i];
            }
            run += own[i];
          }
        }
      }
      __syncthreads();
      top += (uint32_t)found[0] << shift;
      above = found[1];
      members = found[2];
      first = shift;
    } while (shift > 0 && members > kGather);
    const int need = budget - above;  // 1 <= need <= members
    if (shift == 0) {
      equal = members;
    } else {
      // a lane's keys of the bin go to consecutive places
      auto in = [&](uint32_t k) { return k - top < 1u << shift && k - 1u < kSafe - 1u; };
      int mine = 0;
      each([&](int, uint32_t k) { mine += in(k) ? 1 : 0; });
      const int upto = wave_incl_scan(mine, lane);
      int at = 0;
      if (lane == 0) at = atomicAdd(&gathered, wave_last(upto));
      at = __builtin_amdgcn_readfirstlane(at) + upto - mine;
      each([&](int, uint32_t k) {
        if (in(k)) few[at++] = k;
      });
      __syncthreads();
      if (wave == 0) {  // one wave: no barriers between its counts
        constexpr int kOwn = kGather / 64;
        uint32_t own[kOwn];
#pragma unroll
        for (int i = 0; i < kOwn; ++i) own[i] = i * 64 + lane < members ? few[i * 64 + lane] : 0u;
        // (few keys by popcounts of masks; many by a count a lane, as each
        // popcount waits for the scalar unit)
        auto tally = [&](auto f) -> int {
          if (members <= 128) return __popcll(__ballot(f(own[0]))) + __popcll(__ballot(f(own[1])));
          int n = 0;
#pragma unroll
          for (int i = 0; i < kOwn; ++i)
            if (i * 64 < members) n += f(own[i]) ? 1 : 0;
          return wave_last(wave_incl_scan(n, lane));
        };
        for (int bit = (shift + 1) & ~1; bit > 0;) {
          bit -= 2;
          const uint32_t c1 = plus(top, 1u << bit), c2 = plus(top, 2u << bit), c3 = plus(top, 3u << bit);
          if (tally([&](uint32_t k) { return k >= c2; }) >= need)
            top = tally([&](uint32_t k) { return k >= c3; }) >= need ? c3 : c2;
          else if (tally([&](uint32_t k) { return k >= c1; }) >= need)
            top = c1;
        }
        const int same = tally([&](uint32_t k) { return k == top; });
        const int more = tally([&](uint32_t k) { return k > top; });
        if (lane == 0) {
          found[0] = (int)top;
          found[1] = above + more;
          found[2] = same;
        }
      }
      __syncthreads();
      top = (uint32_t)found[0];
      above = found[1];
      equal = found[2];
    }
  }
  // of the keys equal to it, the lowest indices are kept
  const int want = budget - above;
  const bool ties = want < equal;
  int eq = 0;
  if (ties) {
    int mine = 0;
    each([&](int, uint32_t k) { mine += __popcll(__ballot(k == top)); });
    eq = before_and_all<WAVES>(counts[1], mine, wave).x;
  }
  auto kept_of = [&](uint32_t k) {
    if (!ties) return k >= top;
    const uint64_t em = __ballot(k == top);
    const bool kept = k > top || (k == top && eq + rank_in(em) < want);
    eq += __popcll(em);
    return kept;
  };

  if constexpr (E > 0) {
    // One bit an index, and the kept ones before each word of 64: a hole's rank
    // is its index less the kept ones before it.
    constexpr int kWords = THREADS * E / 64;
    __shared__ uint64_t mask[kWords];
    __shared__ int before[kWords];
    __shared__ uint16_t list[THREADS * E / 2];  // at most half of the indices are movers
    static_assert(THREADS * E <= 65536 && kWords <= THREADS, "indices of 16 bits, a word a thread");
    uint32_t word_lo = 0u, word_hi = 0u;  // lane e: the wave's word e
#pragma unroll
    for (int e = 0; e < E; ++e) {
      if (e < items) {
        const uint64_t m = __ballot(kept_of(reg[e]));
        word_lo = lane == e ? (uint32_t)m : word_lo;
        word_hi = lane == e ? (uint32_t)(m >> 32) : word_hi;
      }
    }
    if (lane < items) mask[wave * items + lane] = (uint64_t)word_hi << 32 | word_lo;
    __syncthreads();
    const int filled = WAVES * items;
    const int mine = (int)threadIdx.x < filled ? __popcll(mask[threadIdx.x]) : 0;
    const int upto = wave_incl_scan(mine, lane);
    const int base0 = before_and_all<WAVES>(counts[2], wave_last(upto), wave).x;
    if ((int)threadIdx.x < filled) before[threadIdx.x] = base0 + upto - mine;
    __syncthreads();
    const int words = (len + 63) >> 6, edge = budget >> 6;
    const uint64_t low = (1ull << (budget & 63)) - 1;  // of word `edge`, the slots below budget
    const int below = before[edge] + __popcll(mask[edge] & low);  // kept where they are
    constexpr int kAhead = 4;  // words read ahead of the writes
    for (int w0 = edge + wave; w0 < words; w0 += WAVES * kAhead) {
      uint64_t m[kAhead];
      int at[kAhead];
#pragma unroll
      for (int i = 0; i < kAhead; ++i) {
        const int w = min(w0 + i * WAVES, words - 1);
        m[i] = w0 + i * WAVES < words ? mask[w] : 0;
        at[i] = before[w] - below;
      }
#pragma unroll
      for (int i = 0; i < kAhead; ++i) {
        const int idx = (w0 + i * WAVES) * 64 + lane;
        if (((m[i] >> lane) & 1) != 0 && idx >= budget) list[at[i] + rank_in(m[i])] = (uint16_t)idx;
      }
    }
    __syncthreads();
    for (int w = wave; w * 64 < budget; w += WAVES) {
      const uint64_t m = mask[w];
      const int i = w * 64 + lane;
      if (i < budget) keep[i] = ((m >> lane) & 1) != 0 ? i : (int)list[i - before[w] - rank_in(m)];
    }
  } else {
    // holes and movers of the waves before this one
    __shared__ int list[kListCap];
    const int eq0 = eq;
    auto each_kept = [&](auto f) {
      eq = eq0;
      each([&](int i, uint32_t k) { f(i, kept_of(k)); });
    };
    int holes = 0, movers = 0;
    each_kept([&](int i, bool kept) {
      holes += __popcll(__ballot(i < budget && !kept));
      movers += __popcll(__ballot(i >= budget && kept));
    });
    const int hole0 = before_and_all<WAVES>(counts[2], holes, wave).x;
    const int2 mv = before_and_all<WAVES>(counts[0], movers, wave);
    // they meet in LDS, kListCap at a time
    for (int at = 0; at == 0 || at < mv.y; at += kListCap) {
      int r = mv.x - at;
      each_kept([&](int i, bool kept) {
        const bool mover = i >= budget && kept;
        const uint64_t mm = __ballot(mover);
        const int mine = r + rank_in(mm);
        if (mover && mine >= 0 && mine < kListCap) list[mine] = i;
        r += __popcll(mm);
      });
      __syncthreads();
      r = hole0 - at;
      each_kept([&](int i, bool kept) {
        const bool hole = i < budget && !kept;
        const uint64_t hm = __ballot(hole);
        const int mine = r + rank_in(hm);
        if (hole && mine >= 0 && mine < kListCap) keep[i] = list[mine];
        if (i < budget && kept && at == 0) keep[i] = i;
        r += __popcll(hm);
      });
      __syncthreads();
    }
  }
}

// ---- move --------------------------------------------------------------------
//
// A workgroup looks 256 slots up, moves their weights and positions with a lane
// a slot, and lists the slots that move.  Rows whose channels are contiguous move
// as 16-byte pieces.  Where a channel's tokens are contiguous (channel-major V) a
// row is D single elements; when many of the 256 move, as when a prompt is cut, a
// lane takes a channel of a 16-token run instead and writes the run whole.
constexpr int kSlots = 256;
constexpr int kRuns = kSlots / 16;
// (2,048 slots of 16 sequences and 8 heads of 128 in bf16, of 256 slots 51, 93
// and 128 moving: element by element 34, 51 and 86 us, by runs 68, 70 and 74; in
// e4m3 25, 34 and 46 against 36, 37 and 37.)
constexpr int kTileMoves = 112;

enum MoveMode : int { kRows = 0, kTile = 1, kElements = 2 };

// A cache's strides, by value (pointers into the kernel's arguments would put
// them into scratch memory).
struct Strides {
  int64_t block, token, head, channel;
  // Element offset of a slot, without head and channel.
  __device__ __forceinline__ int64_t slot(int blk, int off) const { return (int64_t)blk * block + (int64_t)off * token; }
};
template <int WHICH>
__device__ __forceinline__ Strides strides_of(const EvictMoveParams& p) {
  return Strides{p.c_s[WHICH][0], p.c_s[WHICH][1], p.c_s[WHICH][2], p.c_s[WHICH][3]};
}

// Slot j of sequence b, account head h: its source, and where both lie.
struct MoveSlot {
  int src_blk, src_off, dst_blk, dst_off;
  bool moved;
};

// Looks slot j up and, with `account`, moves its weight and position.
__device__ __forceinline__ MoveSlot move_slot(const EvictMoveParams& p, int b, int h, int j, bool account) {
  MoveSlot m{0, 0, 0, 0, false};
  // (a source outside the tables cannot come from a selection)
  const int cap = min(p.Mb * p.bs, p.S);
  if (j >= min(p.budget, cap)) return m;
  const int src = p.keep[(int64_t)b * p.k_sb + (int64_t)h * p.k_sh + j];
  if (src < 0 || src >= cap) return m;
  if (account && p.positions != nullptr) {
    const int kept = p.kept[(int64_t)b * p.kept_s];
    if (src != j || j >= kept) {
      const int raw = p.lens[(int64_t)b * p.l_s], len = raw < 0 ? 0 : (raw < p.S ? raw : p.S);
      int32_t* pos = p.positions + (int64_t)b * p.p_sb + (int64_t)h * p.p_sh;
      pos[j] = src < kept ? pos[src] : p.seen[(int64_t)b * p.seen_s] - len + src;
    }
  }
  if (src == j) return m;
  if (account && p.weights != nullptr) {
    float* a = p.weights + (int64_t)b * p.w_sb + (int64_t)h * p.w_sh;
    a[j] = a[src];
  }
  const int32_t* t = p.tables + (int64_t)b * p.t_sb;
  const int jb = (int)((uint32_t)j / (uint32_t)p.bs), sb = (int)((uint32_t)src / (uint32_t)p.bs);
  m.dst_blk = t[(int64_t)jb * p.t_sm];
  m.src_blk = t[(int64_t)sb * p.t_sm];
  m.dst_off = j - jb * p.bs;
  m.src_off = src - sb * p.bs;
  m.moved = m.dst_blk >= 0 && m.dst_blk < p.NB && m.src_blk >= 0 && m.src_blk < p.NB;
  return m;
}

__device__ __forceinline__ int lane_value(int v, int lane) { return __builtin_amdgcn_readlane(v, lane); }

// (the compiler keeps arrays of uint4 that are stored under a condition in
// scratch memory, and arrays of this in registers)
typedef uint32_t Bytes16 __attribute__((ext_vector_type(4)));

// kN pieces a thread of the listed rows' `total` from `from` on, by pieces
// (E = Bytes16) or elements; past the end the last one again, not stored.
template <int kN, class E, class T>
__device__ __forceinline__ void copy_pieces(const Strides& s, T* base, int h0, int per, int row, const int4* list,
                                            int from, int total) {
  constexpr int kElems = (int)(sizeof(E) / sizeof(T));
  E v[kN];
  T* to[kN];
#pragma unroll
  for (int i = 0; i < kN; ++i) {
    const uint32_t u = (uint32_t)min(from + i * 256 + (int)threadIdx.x, total - 1);
    const uint32_t k = u / (uint32_t)row, r = u - k * (uint32_t)row;
    const uint32_t hh = r / (uint32_t)per, c = r - hh * (uint32_t)per;
    const int4 m = list[k];
    const int64_t at = (int64_t)(h0 + (int)hh) * s.head + (int64_t)(c * kElems) * s.channel;
    v[i] = *(const E*)(base + s.slot(m.x, m.y) + at);
    to[i] = base + s.slot(m.z, m.w) + at;
  }
#pragma unroll
  for (int i = 0; i < kN; ++i)
    if (from + i * 256 + (int)threadIdx.x < total) *(E*)to[i] = v[i];
}

// The listed rows of heads [h0, h0 + nh): four pieces a thread in flight, the
// rest two at a time (a few moves must not load four).
template <int WHICH, class E, class T>
__device__ __forceinline__ void copy_listed(const EvictMoveParams& p, int h0, int nh, const int4* list, int n) {
  constexpr int kElems = (int)(sizeof(E) / sizeof(T));
  const Strides s = strides_of<WHICH>(p);
  T* base = (T*)p.cache[WHICH];
  const int per = p.D / kElems, row = nh * per, total = n * row;
  int from = 0;
  for (; from + 4 * 256 <= total; from += 4 * 256)
    copy_pieces<4, E, T>(s, base, h0, per, row, list, from, total);
  for (; from < total; from += 2 * 256) copy_pieces<2, E, T>(s, base, h0, per, row, list, from, total);
}

// Channel-major V of heads [h0, h0 + nh) by runs of 16 slots in which some move:
// a wave takes 64 channels of a run, a lane reads its 16 tokens from where each
// belongs (unmoved ones from their own place: a load that may be left out would
// have to be waited for where the ways meet) and writes them whole.
template <class T>
__device__ __forceinline__ void copy_tiles(const EvictMoveParams& p, int h0, int nh, const int4* slots,
                                           const uint64_t* moved) {
  const Strides s = strides_of<1>(p);
  const int lane = threadIdx.x & 63, parts = (p.D + 63) >> 6, items = nh * kRuns * parts;
  for (int u = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6); u < items; u += 4) {
    const int run = u & (kRuns - 1), hp = u / kRuns, hh = hp / parts, d = (hp - hh * parts) * 64 + lane;
    const uint32_t bits = (uint32_t)__builtin_amdgcn_readfirstlane((int)(moved[run >> 2] >> (run & 3) * 16)) & 0xFFFFu;
    if (bits == 0u) continue;
    const int4 m = slots[run * 16 + (lane & 15)];
    const int l0 = __builtin_ctz(bits);
    // the place of the run's slot 0, from the first that moves
    const int64_t first = s.slot(lane_value(m.z, l0), lane_value(m.w, l0) - l0);
    const int64_t own = (bits >> (lane & 15)) & 1u ? s.slot(m.x, m.y) : first + (lane & 15);
    const int lo = (int)own, hi = (int)(own >> 32);
    // (lanes past the last channel read it again: every lane stays for the shuffles)
    T* base = (T*)p.cache[1] + (int64_t)(h0 + hh) * s.head + (int64_t)min(d, p.D - 1) * s.channel;
    T e[16];
#pragma unroll
    for (int i = 0; i < 16; ++i)
      e[i] = base[(int64_t)((uint64_t)(uint32_t)lane_value(hi, i) << 32 | (uint32_t)lane_value(lo, i))];
    union {
      uint4 q[sizeof(T)];
      T e[16];
    } r;
#pragma unroll
    for (int i = 0; i < 16; ++i) r.e[i] = e[i];
    if (d < p.D) {
#pragma unroll
      for (int i = 0; i < (int)sizeof(T); ++i) ((uint4*)(base + first))[i] = r.q[i];
    }
  }
}

// kSlots slots a workgroup; any strides.
template <class T>
__global__ __launch_bounds__(256) void evict_move_kernel(EvictMoveParams p) {
  __shared__ int4 list[kSlots];  // source block and offset, destination block and offset of the slots that move
  __shared__ int4 slots[kSlots];  // the same by slot
  __shared__ uint64_t moved[4];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int per = (p.budget + kSlots - 1) / kSlots;
  const int bh = blockIdx.x / per, b = bh / p.Hw, h = bh - b * p.Hw;
  const MoveSlot m = move_slot(p, b, h, (int)(blockIdx.x - bh * per) * kSlots + (int)threadIdx.x, true);
  const uint64_t bits = __ballot(m.moved);
  if (lane == 0) moved[wave] = bits;
  __syncthreads();
  int at = 0, n = 0;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int count = __popcll(moved[i]);
    at += i < wave ? count : 0;
    n += count;
  }
  if (n == 0) return;
  const int4 x = make_int4(m.src_blk, m.src_off, m.dst_blk, m.dst_off);
  if (m.moved) list[at + rank_in(bits)] = x;
  slots[threadIdx.x] = x;
  __syncthreads();
  const int nh = p.Hw == 1 ? p.Hkv : 1, h0 = p.Hw == 1 ? 0 : h;
  if (p.mode[0] == kRows) copy_listed<0, Bytes16, T>(p, h0, nh, list, n);
  else copy_listed<0, T, T>(p, h0, nh, list, n);
  if (p.mode[1] == kRows) copy_listed<1, Bytes16, T>(p, h0, nh, list, n);
  else if (p.mode[1] == kTile && n >= kTileMoves) copy_tiles<T>(p, h0, nh, slots, moved);
  else copy_listed<1, T, T>(p, h0, nh, list, n);
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
  // Few threads with many keys leave room for other heads' workgroups, many
  // with few shorten a lone one's chain.  64 sequences of 8 heads without
  // positions (with them), <threads, keys>: 2,064 slots 12.4 us (13.6) on <256, 16>,
  // 12.9 (14.0) on <512, 16>, 22.6 (24.4) on <1024, 16>; 8,000 slots 20.7 (24.7) on
  // <512, 16>, 32.5 (37.2) on <1024, 16> (four sequences: 15.4 and 15.8); 16,000
  // slots 40.6 (49.8) on <1024, 16>, 49.4 (67.9) on <512, 32>.
  if (p.S <= 256 * 4) return launch_select_t<256, 4>(p, stream);
  if (p.S <= 256 * 16) return launch_select_t<256, 16>(p, stream);
  if (p.S <= 512 * 16) return launch_select_t<512, 16>(p, stream);
  if (p.S <= 1024 * 16) return launch_select_t<1024, 16>(p, stream);
  if (p.S <= 1024 * 32) return launch_select_t<1024, 32>(p, stream);
  return launch_select_t<1024, 0>(p, stream);
}

int32_t launch_evict_move(const EvictMoveParams& q, int elem_bytes, hipStream_t stream) {
  EvictMoveParams p = q;
  for (int c = 0; c < 2; ++c) {
    const int64_t* s = p.c_s[c];
    auto whole = [&](int64_t stride) { return (stride * elem_bytes) % 16 == 0; };
    const bool base = ((uintptr_t)p.cache[c] & 15) == 0 && whole(s[0]) && whole(s[2]);
    if (base && s[3] == 1 && whole(s[1]) && whole(p.D)) p.mode[c] = kRows;
    else if (base && s[1] == 1 && whole(s[3]) && p.bs % 16 == 0) p.mode[c] = kTile;
    else p.mode[c] = kElements;
  }
  ProfileScope prof("cf_evict_move", stream);
  const dim3 grid((unsigned)(ceil_div(p.budget, kSlots) * p.Hw * p.B));
  switch (elem_bytes) {
    case 1: CF_LAUNCH((evict_move_kernel<uint8_t>), grid, dim3(256), 0, stream, p); break;
    case 2: CF_LAUNCH((evict_move_kernel<uint16_t>), grid, dim3(256), 0, stream, p); break;
    default: CF_LAUNCH((evict_move_kernel<uint32_t>), grid, dim3(256), 0, stream, p); break;
  }
  CF_HIP_CHECK(hipGetLastError());
  return CF_OK;
}

}  // namespace cf
