// Moves of whole blocks over several paged tensors at once.
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

#include <vector>

namespace cf {

// Steps of a plan: block dst takes what block src holds; src -1: what the group's
// first step set aside; dst -1: src is set aside.
struct MoveStep {
  int32_t src, dst;
};

// Simultaneous moves as steps that can be taken one after the other.  The steps of
// a chain depend on each other and keep their order; chains are independent.
// `whole`: lengths of runs of steps that stay together in a launch (a cycle's share
// the value set aside), in order, per chain.
struct MoveChain {
  std::vector<MoveStep> steps;
  std::vector<int32_t> whole;
};

constexpr int kMaxMoveSteps = 320;   // of a launch
constexpr int kMaxMoveCaches = 16;   // of a launch
constexpr int kMaxCycleSteps = 256;  // a longer cycle is taken in parts

// moves [n][2] = (source, destination), each destination once.
std::vector<MoveChain> plan_moves(const int32_t* moves, int64_t n);

}  // namespace cf
