// Blocks of several paged tensors copied or rearranged: block dst_i takes what
// block src_i held before the call.
//
// A source may go to several destinations, and a destination may be the source of
// another move, so the moves are a graph in which every block has one way in.  Its
// components are trees (copies, and chains of blocks that each make room for the
// next) and cycles with trees on them.  The host orders each: a block is written
// only after every move out of it, and a cycle starts by setting its first block
// aside in a register.  On the device a thread takes the same 16 bytes of every
// block of a component, step by step, so nothing is shared between threads: no
// barrier, no memory for what is set aside, and a chain of any length is one pass.
// The loads of kAhead steps go out before their stores (a load reads what was there
// before the call, so it may be early).
//
// The steps and the tensors are kernel arguments: nothing is uploaded, and a
// captured call replays with the moves it was given.  A chain costs a word a block.
//
// Bound by HBM.  A component's steps are one after the other, so the bytes in flight
// are those of one block over all tensors, times kAhead and the components at hand.
// 1,800 blocks of 256 KiB (945 MB read and written): in 220 chains of up to 35 blocks,
// as a fragmented pool is compacted, 215 us, 4.4 TB/s of the 4.8 that a large copy
// reaches; in one chain 211 us, in one cycle 219, in eight 232.  With 8 steps ahead and
// 8 bytes of arguments a step the first took 520.  16 copies of 1 MiB: 8.2 us.
//
// STRETCH (a launch with a run of more than two batches' words): batches of one chain
// take a way of their own without a test a step, which the one chain needs (476 us
// without it).  It holds 208 VGPRs instead of 144, and the 16 copies take 11.4 us in it.
#include <algorithm>
#include <numeric>

#include "cf_device.hpp"
#include "cf_host.hpp"
#include "move_blocks.hpp"

namespace cf {

namespace {

constexpr int kAhead = 32;
// Workgroups have 256 threads, or 64 where that makes fewer than so many: a long chain
// over few tensors then takes all CUs.
constexpr int kFewGroups = 512;
constexpr int kMoveShapes = 4;    // tensors of a launch differ in at most so many shapes
constexpr int kMoveCaches = 128;  // tensors of a launch
constexpr int kMoveLists = 32;    // lists of steps that run side by side
constexpr int kMoveGroups = 65536;  // workgroups of a tensor
constexpr int kMoveWords = 952;   // words of a launch: tensors, lists' starts and blocks
constexpr uint32_t kLastBlock = 1u << 31;
constexpr uint32_t kAside = kLastBlock - 1;  // in a block's place: the value set aside

struct MoveShape {
  int64_t stride, bytes;  // between blocks, of a block
  int32_t unit;           // bytes a thread moves: 16, 4 or 1
  int32_t groups;         // workgroups of a tensor (their threads take further pieces in a loop)
  int32_t first_group, first_cache;
};

// words: the tensors' addresses (two each), the first block of each list and the end
// of the last, then the lists: paths of blocks, the last one's word marked.
struct MoveArgs {
  MoveShape shape[kMoveShapes];
  int32_t caches, lists;
  uint32_t word[kMoveWords + kAhead + 1];  // (read in whole batches, past the end too)
};
static_assert(sizeof(MoveArgs) <= 4096, "kernel arguments");

template <class T, bool STRETCH>
__device__ __forceinline__ void move_pieces(const uint32_t* __restrict__ word, int begin, int end, char* base,
                                            const MoveShape& sh, int group) {
  const int64_t pieces = sh.bytes / (int64_t)sizeof(T), stride = sh.stride / (int64_t)sizeof(T);
  for (int64_t i = (int64_t)group * blockDim.x + threadIdx.x; i < pieces; i += (int64_t)sh.groups * blockDim.x) {
    T* at = (T*)base + i;
    T aside{};
    for (int e = begin; e < end; e += kAhead) {
      uint32_t w[kAhead + 1];
#pragma unroll
      for (int u = 0; u <= kAhead; ++u) w[u] = word[e + u];
      T v[kAhead];
      if constexpr (STRETCH) {
        // a stretch of one chain, without ends and what is set aside
        uint32_t most = 0;
#pragma unroll
        for (int u = 0; u <= kAhead; ++u) most = max(most, w[u]);
        if (most < kAside && e + kAhead < end && sh.bytes < (int64_t)1 << 32) {
          const uint32_t off = (uint32_t)i * (uint32_t)sizeof(T);
#pragma unroll
          for (int u = 0; u < kAhead; ++u) v[u] = *(const T*)(base + (uint64_t)w[u + 1] * (uint64_t)sh.stride + off);
#pragma unroll
          for (int u = 0; u < kAhead; ++u) *(T*)(base + (uint64_t)w[u] * (uint64_t)sh.stride + off) = v[u];
          continue;
        }
      }
#pragma unroll
      for (int u = 0; u < kAhead; ++u) {
        const uint32_t src = w[u + 1] & ~kLastBlock;
        v[u] = T{};
        if (e + u < end && !(w[u] & kLastBlock) && src != kAside) v[u] = at[src * stride];
      }
#pragma unroll
      for (int u = 0; u < kAhead; ++u) {
        if (e + u < end && !(w[u] & kLastBlock)) {
          const T x = (w[u + 1] & ~kLastBlock) == kAside ? aside : v[u];
          if (w[u] == kAside) aside = x;
          else at[w[u] * stride] = x;
        }
      }
    }
  }
}

template <bool STRETCH>
__global__ __launch_bounds__(256) void move_blocks_kernel(MoveArgs a) {
  int k = 0;
  while (k + 1 < kMoveShapes && (int)blockIdx.x >= a.shape[k + 1].first_group) ++k;
  const MoveShape sh = a.shape[k];
  const int at = (int)blockIdx.x - sh.first_group, c = at / sh.groups, group = at - c * sh.groups;
  char* base = (char*)((uint64_t)a.word[2 * (sh.first_cache + c)] | (uint64_t)a.word[2 * (sh.first_cache + c) + 1] << 32);
  const uint32_t* lists = a.word + 2 * a.caches + blockIdx.y;
  const int begin = (int)lists[0], end = (int)lists[1];
  if (sh.unit == 16) move_pieces<uint4, STRETCH>(a.word, begin, end, base, sh, group);
  else if (sh.unit == 4) move_pieces<uint32_t, STRETCH>(a.word, begin, end, base, sh, group);
  else move_pieces<uint8_t, STRETCH>(a.word, begin, end, base, sh, group);
}

}  // namespace

std::vector<MoveComponent> plan_moves(const int32_t* moves, int64_t n, int64_t blocks) {
  struct Move {
    int32_t src, dst;
  };
  std::vector<Move> m;
  m.reserve(n);
  for (int64_t i = 0; i < n; ++i)
    if (moves[2 * i] != moves[2 * i + 1]) m.push_back(Move{moves[2 * i], moves[2 * i + 1]});
  std::vector<int32_t> into(blocks, -1);  // the move into a block
  for (size_t i = 0; i < m.size(); ++i) into[m[i].dst] = (int32_t)i;
  // waits[i]: the move that overwrites i's source, which has to wait for i
  std::vector<int32_t> waits(m.size(), -1), pending(m.size(), 0), group(m.size());
  std::iota(group.begin(), group.end(), 0);
  auto root = [&](int32_t i) {
    while (group[i] != i) i = group[i] = group[group[i]];
    return i;
  };
  for (size_t i = 0; i < m.size(); ++i) {
    const int32_t next = into[m[i].src];
    if (next < 0) continue;
    waits[i] = next;
    ++pending[next];
    group[root((int32_t)i)] = root(next);
  }
  // components in the order of their first move
  std::vector<MoveComponent> all;
  std::vector<int32_t> index(m.size(), -1);
  auto component = [&](int32_t i) -> MoveComponent& {
    int32_t& c = index[root(i)];
    if (c < 0) {
      c = (int32_t)all.size();
      all.emplace_back();
    }
    return all[c];
  };
  std::vector<char> done(m.size(), 0);
  for (size_t i = 0; i < m.size(); ++i) {
    // a move that nothing waits behind, then the one it made room for, and so on
    if (done[i] || pending[i] != 0) continue;
    MovePath path{{m[i].dst}, false};
    for (int32_t k = (int32_t)i; k >= 0 && !done[k] && pending[k] == 0;) {
      path.blocks.push_back(m[k].src);
      done[k] = 1;
      k = waits[k];
      if (k >= 0) --pending[k];
    }
    component((int32_t)i).push_back(std::move(path));
  }
  for (size_t i = 0; i < m.size(); ++i) {
    if (done[i]) continue;
    // what is left are cycles: d0 <- d1 <- ... <- d0
    MovePath path{{}, true};
    for (int32_t k = (int32_t)i; !done[k]; k = waits[k]) {
      done[k] = 1;
      path.blocks.push_back(m[k].dst);
    }
    component((int32_t)i).push_back(std::move(path));
  }
  return all;
}

namespace {

struct MoveCache {
  char* base;
  int64_t stride, bytes;
  int64_t blocks;

  const char* end() const { return base + (blocks - 1) * stride + bytes; }
};

// b begins where a does or behind it.
bool share_bytes(const MoveCache& a, const MoveCache& b) {
  if (a.stride == b.stride) {
    // b's first block begins in a's block k's share of the stride
    const int64_t k = (b.base - a.base) / a.stride, in = (b.base - a.base) % a.stride;
    return (k < a.blocks && in < a.bytes) || (k + 1 < a.blocks && a.stride - in < b.bytes);
  }
  for (int64_t i = 0, j = 0; i < a.blocks && j < b.blocks;) {
    const char *x = a.base + i * a.stride, *y = b.base + j * b.stride;
    if (x + a.bytes <= y) ++i;
    else if (y + b.bytes <= x) ++j;
    else return true;
  }
  return false;
}

// Whether some of the tensors, in order of their addresses, share bytes.  Those whose
// ranges meet are mostly slices of one slab (layers, K's and V's scales), with one
// stride: apart if they are within it, which a sort of their places there tells; what
// that does not settle is compared block by block.
bool any_share_bytes(const std::vector<MoveCache>& caches) {
  std::vector<std::pair<int64_t, int64_t>> places;  // within the stride: first byte, past the last
  for (size_t c = 0; c < caches.size();) {
    const size_t first = c;
    const int64_t stride = caches[c].stride;
    const char* end = caches[c].end();
    bool one_stride = true;
    for (++c; c < caches.size() && caches[c].base < end; ++c) {
      end = std::max(end, caches[c].end());
      one_stride = one_stride && caches[c].stride == stride;
    }
    if (c - first == 1) continue;
    if (one_stride) {
      places.clear();
      for (size_t k = first; k < c; ++k) {
        const int64_t at = (caches[k].base - caches[first].base) % stride;
        places.emplace_back(at, at + caches[k].bytes);
      }
      std::sort(places.begin(), places.end());
      bool apart = places.back().second <= stride + places.front().first;
      for (size_t k = 1; k < places.size(); ++k) apart = apart && places[k - 1].second <= places[k].first;
      if (apart) continue;
    }
    for (size_t k = first; k < c; ++k)
      for (size_t o = k + 1; o < c; ++o)
        if (share_bytes(caches[k], caches[o])) return true;
  }
  return false;
}

// The steps of a component that no launch has taken yet.
struct MoveRest {
  const MoveComponent* paths;
  size_t path = 0, at = 0;  // at: blocks of the path that are done with
  int64_t words = 0;

  explicit MoveRest(const MoveComponent& c) : paths(&c) {
    for (const MovePath& p : c) words += cost(p, 0);
  }
  // A path's words from block `from` on: a cycle sets a block aside and back.
  static int64_t cost(const MovePath& p, size_t from) { return (int64_t)(p.blocks.size() - from) + (p.cycle ? 2 : 0); }
  bool done() const { return path == paths->size(); }
  // Appends at most `room` words of steps to a launch's list.
  void take(int64_t room, std::vector<uint32_t>& list) {
    while (!done()) {
      const MovePath& p = (*paths)[path];
      const int64_t whole = cost(p, at), least = p.cycle ? 4 : 2;
      if (room < std::min(whole, least)) return;
      const size_t n = whole <= room ? p.blocks.size() - at : (size_t)(room - (p.cycle ? 2 : 0));
      if (p.cycle) list.push_back(kAside);
      for (size_t k = at; k < at + n; ++k) list.push_back((uint32_t)p.blocks[k]);
      if (p.cycle) list.push_back(kAside);
      list.back() |= kLastBlock;
      words -= whole;
      if (at + n == p.blocks.size()) {
        room -= whole;
        ++path;
        at = 0;
      } else {
        // The last block taken is the first of what is left.  In a cycle it holds the
        // first one's value in between and is read again, in a later launch: steps of
        // one launch read ahead.
        at += n - 1;
        words += cost(p, at);
        return;
      }
    }
  }
};

// Deals the tensors' pieces to workgroups of so many threads; returns their number.
int64_t deal_groups(MoveArgs& a, int threads) {
  int64_t groups = 0;
  for (int k = 0; k < kMoveShapes; ++k) {
    MoveShape& s = a.shape[k];
    const int last = k + 1 < kMoveShapes ? a.shape[k + 1].first_cache : a.caches;
    s.first_group = (int32_t)groups;
    if (s.unit == 0) {
      s.first_group = INT32_MAX;  // no such shape
      continue;
    }
    s.groups = (int32_t)std::min<int64_t>(ceil_div(s.bytes / s.unit, threads), kMoveGroups);
    groups += (int64_t)s.groups * (last - s.first_cache);
  }
  return groups;
}

int32_t launch_moves(const std::vector<MoveComponent>& plan, MoveArgs& a, hipStream_t stream) {
  // Lists enough for 16 waves on every SIMD, of at least kAhead / 2 words: 16 copies
  // of 1 MiB take 8.9 us in one list, 8.7 in 2, 11.0 in 4 and 20.7 in 16; chains of
  // hundreds of blocks 94 us a launch in up to 32, 98 in up to 20, 104 in up to 8.
  constexpr int64_t kThreads = 1024 * 1024;
  const int64_t most = std::min<int64_t>(ceil_div(kThreads, deal_groups(a, 256) * 256), kMoveLists);
  const int64_t room = kMoveWords - 2 * a.caches - (kMoveLists + 1);
  constexpr int64_t kLong = 64;  // words of a component that may be cut
  std::vector<MoveRest> cut, whole;
  int64_t all = 0;
  for (const MoveComponent& c : plan) {
    MoveRest r(c);
    all += r.words;
    (r.words > kLong ? cut : whole).push_back(r);
  }
  std::sort(cut.begin(), cut.end(), [](const MoveRest& x, const MoveRest& y) { return x.words > y.words; });
  for (size_t next = 0; next < whole.size() || !cut.empty();) {
    // every long component its share of each of the launches that all need, and
    // others as they come
    int64_t left = room;
    const int64_t launches = ceil_div(all, room);
    std::vector<std::vector<uint32_t>> runs;
    auto take = [&](MoveRest& r, int64_t most_words) {
      std::vector<uint32_t> run;
      const int64_t before = r.words;
      r.take(most_words, run);
      all -= before - r.words;
      left -= (int64_t)run.size();
      if (!run.empty()) runs.push_back(std::move(run));
    };
    for (MoveRest& r : cut) {
      if (left < kLong) break;
      take(r, std::min(left, launches == 1 ? left : std::max(ceil_div(r.words, launches) + 2, kLong)));
    }
    cut.erase(std::remove_if(cut.begin(), cut.end(), [](const MoveRest& r) { return r.done(); }), cut.end());
    for (; next < whole.size() && whole[next].words <= left; ++next) take(whole[next], left);
    // the longest run to the shortest list
    std::sort(runs.begin(), runs.end(), [](const auto& x, const auto& y) { return x.size() > y.size(); });
    const int64_t wanted = std::max<int64_t>(1, std::min(most, 2 * (room - left) / kAhead));
    std::vector<std::vector<uint32_t>> lists(std::min<size_t>(runs.size(), (size_t)wanted));
    for (const auto& run : runs) {
      auto& to = *std::min_element(lists.begin(), lists.end(), [](const auto& x, const auto& y) { return x.size() < y.size(); });
      to.insert(to.end(), run.begin(), run.end());
    }
    a.lists = (int32_t)lists.size();
    uint32_t* first = a.word + 2 * a.caches;
    uint32_t at = (uint32_t)(2 * a.caches + a.lists + 1);
    for (size_t l = 0; l < lists.size(); ++l) {
      first[l] = at;
      for (const uint32_t w : lists[l]) a.word[at++] = w;
    }
    first[a.lists] = at;
    const int threads = deal_groups(a, 256) * a.lists < kFewGroups ? 64 : 256;
    const dim3 grid((unsigned)deal_groups(a, threads), (unsigned)a.lists);
    ProfileScope prof("cf_move_blocks", stream);
    if (runs.front().size() > kLong) CF_LAUNCH((move_blocks_kernel<true>), grid, dim3(threads), 0, stream, a);
    else CF_LAUNCH((move_blocks_kernel<false>), grid, dim3(threads), 0, stream, a);
    CF_HIP_CHECK(hipGetLastError());
  }
  return CF_OK;
}

int32_t move_all(std::vector<MoveCache>& caches, const int32_t* moves, int64_t n, int64_t blocks, hipStream_t stream) {
  const std::vector<MoveComponent> plan = plan_moves(moves, n, blocks);
  if (plan.empty()) return CF_OK;
  auto shape = [](const MoveCache& c) { return std::make_pair(c.bytes, c.stride); };
  std::stable_sort(caches.begin(), caches.end(), [&](const auto& x, const auto& y) { return shape(x) > shape(y); });
  auto unit_of = [](const MoveCache& c) {
    const uint64_t all = (uint64_t)(uintptr_t)c.base | (uint64_t)c.stride | (uint64_t)c.bytes;
    return all % 16 == 0 ? 16 : (all % 4 == 0 ? 4 : 1);
  };
  for (size_t c = 0; c < caches.size();) {
    MoveArgs a{};
    int shapes = 0;
    for (; c < caches.size() && a.caches < kMoveCaches; ++c) {
      const int unit = unit_of(caches[c]);
      MoveShape* s = shapes > 0 ? &a.shape[shapes - 1] : nullptr;
      if (s == nullptr || s->bytes != caches[c].bytes || s->stride != caches[c].stride || s->unit != unit) {
        if (shapes == kMoveShapes) break;
        s = &a.shape[shapes++];
        *s = MoveShape{caches[c].stride, caches[c].bytes, unit, 0, 0, a.caches};
      }
      const uint64_t base = (uint64_t)(uintptr_t)caches[c].base;
      a.word[2 * a.caches] = (uint32_t)base;
      a.word[2 * a.caches + 1] = (uint32_t)(base >> 32);
      ++a.caches;
    }
    for (int k = shapes; k < kMoveShapes; ++k) a.shape[k].first_cache = a.caches;
    if (const int32_t rc = launch_moves(plan, a, stream)) return rc;
  }
  return CF_OK;
}

}  // namespace

}  // namespace cf

using namespace cf;

extern "C" int32_t cf_move_blocks(const CfTensor* caches, int32_t n_caches, const int32_t* moves, int64_t n_moves,
                                  void* stream) {
  CF_CHECK(n_caches >= 0 && (n_caches == 0 || caches != nullptr), "caches: NULL or a negative count");
  CF_CHECK(n_moves >= 0 && (n_moves == 0 || moves != nullptr), "moves: NULL or a negative count");
  try {
    std::vector<MoveCache> list;
    int64_t blocks = INT64_MAX;
    for (int32_t c = 0; c < n_caches; ++c) {
      View v;
      const int32_t rc = view_of(&caches[c], "caches", 2, &v);
      if (rc) return rc;
      CF_CHECK(v.stride[1] == 1 || v.size[1] <= 1, "cache %d: each block's elements must be contiguous ([NB, E], E stride 1)",
               c);
      CF_CHECK(v.size[0] <= 1 || v.stride[0] >= v.size[1], "cache %d: blocks overlap", c);
      blocks = std::min(blocks, v.size[0]);
      if (v.size[0] > 0 && v.size[1] > 0) list.push_back(MoveCache{v.base, std::max(v.stride[0], v.size[1]) * v.elem, v.size[1] * v.elem, v.size[0]});
    }
    if (n_caches == 0) return CF_OK;
    std::vector<MoveCache> by_base = list;
    std::sort(by_base.begin(), by_base.end(), [](const MoveCache& x, const MoveCache& y) { return x.base < y.base; });
    CF_CHECK(std::adjacent_find(by_base.begin(), by_base.end(),
                                [](const MoveCache& x, const MoveCache& y) { return x.base == y.base; }) == by_base.end(),
             "one of the caches is given twice");
    CF_CHECK(!any_share_bytes(by_base), "two of the caches share memory");
    CF_CHECK(list.empty() || blocks < INT32_MAX, "caches of %lld blocks are too large", (long long)blocks);
    int64_t most = -1;
    for (int64_t i = 0; i < n_moves; ++i) {
      const int32_t s = moves[2 * i], d = moves[2 * i + 1];
      CF_CHECK(s >= 0 && s < blocks && d >= 0 && d < blocks, "move %lld: block %d or %d is outside the caches' %lld blocks",
               (long long)i, s, d, (long long)blocks);
      most = std::max<int64_t>(most, std::max(s, d));
    }
    std::vector<char> taken(most + 1, 0);
    for (int64_t i = 0; i < n_moves; ++i) {
      CF_CHECK(!taken[moves[2 * i + 1]], "block %d is the destination of two moves", moves[2 * i + 1]);
      taken[moves[2 * i + 1]] = 1;
    }
    if (n_moves == 0 || list.empty()) return CF_OK;
    return move_all(list, moves, n_moves, most + 1, (hipStream_t)stream);
  } catch (...) {
    set_error("cf_move_blocks: out of host memory");
    return CF_ERR_INVALID;
  }
}
