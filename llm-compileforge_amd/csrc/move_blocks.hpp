// Moves of whole blocks over several paged tensors at once.
#pragma once

#include <stdint.h>

#include <vector>

namespace cf {

// Blocks of which each takes what the next one holds, from the first on; in a cycle
// the last takes what the first one held.
struct MovePath {
  std::vector<int32_t> blocks;
  bool cycle;
};

// Simultaneous moves as paths that can be taken one after the other: those of a
// component depend on each other and keep their order, components are independent.
using MoveComponent = std::vector<MovePath>;

// moves [n][2] = (source, destination) of blocks [0, blocks), each destination once.
std::vector<MoveComponent> plan_moves(const int32_t* moves, int64_t n, int64_t blocks);

}  // namespace cf
