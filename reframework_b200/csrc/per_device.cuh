// What a kernel's set-up finds on each device (function attributes and
// occupancy are a device's own).
#pragma once

#include <atomic>

namespace rf {

// A count per device, found once.  Plain C++ without allocation or locks, so
// that nothing is thrown through a C entry: two threads that come first both
// look, and find the same.  A failure (0) is not kept: the next call looks again.
class PerDevice {
 public:
  // `find` looks on device `dev`, the current one.
  template <typename F>
  int get(int dev, F find) {
    if (dev < 0) return 0;
    if (dev >= DEVICES) return find();
    int n = found_[dev].load(std::memory_order_acquire);
    if (n > 0) return n;
    n = find();
    if (n > 0) found_[dev].store(n, std::memory_order_release);
    return n > 0 ? n : 0;
  }

 private:
  static constexpr int DEVICES = 64;
  std::atomic<int> found_[DEVICES] = {};
};

}  // namespace rf
