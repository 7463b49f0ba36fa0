// A setting that has to be made once per device (plain C++, so that it can be tested without a GPU).
#pragma once
#include <atomic>

namespace mlpsp {

// Settings that CUDA keeps per device (the opt-in dynamic shared-memory size of a kernel, for one) must be made once on each device of
// a process.  The caller keeps one DeviceOnce per setting.  A device counts as done only when its setting has been made: host threads whose first calls
// meet all make it, the same one, and none goes on before that; one that failed is made again by the next call.
class DeviceOnce {
 public:
  // set(), which answers 0 for success, unless it has succeeded on this device before.  Devices outside 0 .. 63: every time.
  template <typename Set>
  int apply(int device, Set&& set) {
    const bool known = device >= 0 && device < kDevices;
    if (known && done_[device].load(std::memory_order_acquire)) return 0;
    const int rc = set();
    if (known && rc == 0) done_[device].store(true, std::memory_order_release);
    return rc;
  }

 private:
  static constexpr int kDevices = 64;
  std::atomic<bool> done_[kDevices] = {};
};

}  // namespace mlpsp
