// Arrival counters of launches whose blocks find out who comes last, or wait
// for one another.
//
// Every (device, stream) has two sets, used in turn: a launch counts in one
// and clears the other, which the launch before it left behind.  So it finds
// zeros whatever became of that launch: one whose bounded wait expired ends
// with its counts half way.  Launches of one stream never overlap, and those
// of different streams share nothing.  A captured graph has a set of its own,
// zeroed by the graph.
#pragma once

#include <torch/extension.h>

namespace t1 {

struct Arrivals {
  int* use = nullptr;    // zero at the launch
  int* clear = nullptr;  // counters of the launch before
  int clear_n = 0;
};

__device__ __forceinline__ void clear_arrivals(const Arrivals& a) {
  if (blockIdx.x == 0)
    for (int i = threadIdx.x; i < a.clear_n; i += static_cast<int>(blockDim.x)) a.clear[i] = 0;
}

struct ArrivalSets {
  torch::Tensor counters;  // two sets of `capacity`
  int64_t capacity = 0, used = 0;  // counters that the last launch had
  int next = 0;
};

// n counters for one launch on the current stream; launched() once it is
// under way, so that one that was refused changes nothing.
class ArrivalCounters {
 public:
  explicit ArrivalCounters(int64_t n);
  void launched() {
    if (sets_ == nullptr) return;
    sets_->used = n_;
    sets_->next ^= 1;
  }
  Arrivals arrivals;

 private:
  torch::Tensor held_;  // a graph's own
  ArrivalSets* sets_ = nullptr;
  int64_t n_;
};

}  // namespace t1
