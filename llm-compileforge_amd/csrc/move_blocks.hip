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
// captured call replays with the moves it was given.
#include <algorithm>
#include <numeric>
#include <unordered_map>

#include "cf_device.hpp"
#include "cf_host.hpp"
#include "move_blocks.hpp"

namespace cf {

namespace {

constexpr int kAhead = 8;
constexpr int kMoveThreads = 256;

struct MoveCache {
  char* base;
  int64_t stride, bytes;  // between blocks, of a block
};

struct MoveArgs {
  MoveCache cache[kMaxMoveCaches];
  MoveStep step[kMaxMoveSteps];
  uint16_t first[kMaxMoveSteps + 1];  // first step of each chain
  uint8_t unit[kMaxMoveCaches];       // bytes a thread moves: 16, 4 or 1
};
static_assert(sizeof(MoveArgs) <= 4096, "kernel arguments");

template <class T>
__device__ __forceinline__ void move_pieces(const MoveArgs& a, const MoveCache& c) {
  const int begin = a.first[blockIdx.y], end = a.first[blockIdx.y + 1];
  const int64_t pieces = c.bytes / (int64_t)sizeof(T);
  for (int64_t i = (int64_t)blockIdx.x * kMoveThreads + threadIdx.x; i < pieces; i += (int64_t)gridDim.x * kMoveThreads) {
    T* at = (T*)c.base + i;
    const int64_t stride = c.stride / (int64_t)sizeof(T);
    T aside{};
    for (int e = begin; e < end; e += kAhead) {
      T v[kAhead];
#pragma unroll
      for (int u = 0; u < kAhead; ++u) {
        const int s = e + u < end ? a.step[e + u].src : -1;
        v[u] = T{};
        if (s >= 0) v[u] = at[s * stride];
      }
#pragma unroll
      for (int u = 0; u < kAhead; ++u) {
        if (e + u < end) {
          const MoveStep s = a.step[e + u];
          if (s.dst >= 0) at[s.dst * stride] = s.src >= 0 ? v[u] : aside;
          else aside = v[u];
        }
      }
    }
  }
}

__global__ __launch_bounds__(kMoveThreads) void move_blocks_kernel(MoveArgs a) {
  const MoveCache c = a.cache[blockIdx.z];
  const int unit = a.unit[blockIdx.z];
  if (unit == 16) move_pieces<uint4>(a, c);
  else if (unit == 4) move_pieces<uint32_t>(a, c);
  else move_pieces<uint8_t>(a, c);
}

}  // namespace

std::vector<MoveChain> plan_moves(const int32_t* moves, int64_t n) {
  std::vector<MoveStep> m;
  m.reserve(n);
  for (int64_t i = 0; i < n; ++i)
    if (moves[2 * i] != moves[2 * i + 1]) m.push_back(MoveStep{moves[2 * i], moves[2 * i + 1]});
  std::unordered_map<int32_t, int32_t> into;  // destination -> its move
  into.reserve(m.size() * 2);
  for (size_t i = 0; i < m.size(); ++i) into[m[i].dst] = (int32_t)i;
  // into_src[i]: the move that overwrites i's source, which has to wait for i
  std::vector<int32_t> waits(m.size(), -1), pending(m.size(), 0), group(m.size());
  std::iota(group.begin(), group.end(), 0);
  auto root = [&](int32_t i) {
    while (group[i] != i) i = group[i] = group[group[i]];
    return i;
  };
  for (size_t i = 0; i < m.size(); ++i) {
    const auto it = into.find(m[i].src);
    if (it == into.end()) continue;
    waits[i] = it->second;
    ++pending[it->second];
    group[root((int32_t)i)] = root(it->second);
  }
  // chains in the order of their first move
  std::vector<MoveChain> chains;
  std::vector<int32_t> chain_of(m.size(), -1);
  auto chain = [&](int32_t i) -> MoveChain& {
    int32_t& c = chain_of[root(i)];
    if (c < 0) {
      c = (int32_t)chains.size();
      chains.emplace_back();
    }
    return chains[c];
  };
  std::vector<char> done(m.size(), 0);
  for (size_t i = 0; i < m.size(); ++i) {
    // a move that nothing waits behind, then the one it made room for, and so on
    int32_t k = (int32_t)i;
    while (k >= 0 && !done[k] && pending[k] == 0) {
      MoveChain& c = chain(k);
      c.steps.push_back(m[k]);
      c.whole.push_back(1);
      done[k] = 1;
      k = waits[k];
      if (k >= 0) --pending[k];
    }
  }
  for (size_t i = 0; i < m.size(); ++i) {
    if (done[i]) continue;
    // what is left are cycles: d0 <- d1 <- ... <- d0
    std::vector<int32_t> cycle;
    for (int32_t k = (int32_t)i; !done[k]; k = waits[k]) {
      done[k] = 1;
      cycle.push_back(m[k].dst);
    }
    MoveChain& c = chain((int32_t)i);
    // A cycle of d0 ... dk is one of d0 ... dj and then one of dj ... dk: dj holds
    // d0's value in between.
    const size_t len = cycle.size();
    for (size_t at = 0; at + 1 < len;) {
      const size_t last = std::min(len - 1, at + kMaxCycleSteps - 2);
      c.steps.push_back(MoveStep{cycle[at], -1});
      for (size_t k = at; k < last; ++k) c.steps.push_back(MoveStep{cycle[k + 1], cycle[k]});
      c.steps.push_back(MoveStep{-1, cycle[last]});
      c.whole.push_back((int32_t)(last - at) + 2);
      at = last;
    }
  }
  return chains;
}

namespace {

int32_t launch_moves(const MoveArgs& a, int chains, int caches, hipStream_t stream) {
  int64_t most = 1;
  for (int c = 0; c < caches; ++c)
    if (a.unit[c] > 0) most = std::max(most, ceil_div(a.cache[c].bytes / a.unit[c], kMoveThreads));
  // (a thread's loop takes what is beyond the grid)
  const dim3 grid((unsigned)std::min<int64_t>(most, 1024), (unsigned)chains, (unsigned)caches);
  ProfileScope prof("cf_move_blocks", stream);
  CF_LAUNCH(move_blocks_kernel, grid, dim3(kMoveThreads), 0, stream, a);
  CF_HIP_CHECK(hipGetLastError());
  return CF_OK;
}

int32_t move_all(const std::vector<MoveCache>& caches, const int32_t* moves, int64_t n, hipStream_t stream) {
  const std::vector<MoveChain> chains = plan_moves(moves, n);
  for (size_t c0 = 0; c0 < caches.size(); c0 += kMaxMoveCaches) {
    const int nc = (int)std::min<size_t>(kMaxMoveCaches, caches.size() - c0);
    MoveArgs a{};
    for (int c = 0; c < nc; ++c) {
      a.cache[c] = caches[c0 + c];
      const uint64_t all = (uint64_t)(uintptr_t)a.cache[c].base | (uint64_t)a.cache[c].stride | (uint64_t)a.cache[c].bytes;
      a.unit[c] = all % 16 == 0 ? 16 : (all % 4 == 0 ? 4 : 1);
    }
    int steps = 0, count = 0;
    auto flush = [&]() -> int32_t {
      if (count == 0) return CF_OK;
      a.first[count] = (uint16_t)steps;
      const int32_t rc = launch_moves(a, count, nc, stream);
      steps = count = 0;
      return rc;
    };
    for (const MoveChain& ch : chains) {
      size_t at = 0;
      bool open = false;
      for (const int32_t w : ch.whole) {
        if (steps + w > kMaxMoveSteps) {  // the rest of the chain follows on the stream
          if (const int32_t rc = flush()) return rc;
          open = false;
        }
        if (!open) a.first[count++] = (uint16_t)steps;
        open = true;
        for (int32_t k = 0; k < w; ++k) a.step[steps++] = ch.steps[at++];
      }
    }
    if (const int32_t rc = flush()) return rc;
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
      if (v.size[0] > 0 && v.size[1] > 0) list.push_back(MoveCache{v.base, v.stride[0] * v.elem, v.size[1] * v.elem});
    }
    if (n_caches == 0) return CF_OK;
    std::vector<int32_t> to;
    to.reserve(n_moves);
    for (int64_t i = 0; i < n_moves; ++i) {
      const int32_t s = moves[2 * i], d = moves[2 * i + 1];
      CF_CHECK(s >= 0 && s < blocks && d >= 0 && d < blocks, "move %lld: block %d or %d is outside the caches' %lld blocks",
               (long long)i, s, d, (long long)blocks);
      to.push_back(d);
    }
    std::sort(to.begin(), to.end());
    const auto twice = std::adjacent_find(to.begin(), to.end());
    CF_CHECK(twice == to.end(), "block %d is the destination of two moves", twice == to.end() ? 0 : *twice);
    if (n_moves == 0 || list.empty()) return CF_OK;
    return move_all(list, moves, n_moves, (hipStream_t)stream);
  } catch (...) {
    set_error("cf_move_blocks: out of host memory");
    return CF_ERR_INVALID;
  }
}
