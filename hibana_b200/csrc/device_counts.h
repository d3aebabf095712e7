#pragma once
// Numbers that are asked of a device once and kept for the life of the process (how many clusters it holds at a time): one table for each
// device, since kernel attributes are set for each and a device may hold fewer than another. Plain C++: tests compile it on the host.
#include <atomic>

namespace hb {

constexpr int kMaxDevices = 16;   // of a process: kernel attributes are set once on each

template <int N>
class DeviceCounts {
  std::atomic<int> known_[kMaxDevices][N] = {};      // + 1; 0: not known yet

 public:
  // Number `index` of `device`: the stored one, or what `query` answers. A negative answer says that the query failed: that
  // counts as none this time, and the next call asks again.
  template <typename Query>
  int get(int device, int index, Query&& query) {
    std::atomic<int>& slot = known_[device][index];
    if (const int seen = slot.load(std::memory_order_relaxed); seen > 0) return seen - 1;
    const int n = query();
    if (n < 0) return 0;
    slot.store(n + 1, std::memory_order_relaxed);     // (threads that ask at once store the same number)
    return n;
  }
};

}  // namespace hb
