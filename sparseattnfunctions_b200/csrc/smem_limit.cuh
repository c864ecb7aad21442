// smem_limit.cuh -- a kernel's dynamic shared memory limit per device, raised
// by whichever launch first needs more.  Plain C++ (no CUDA types).
#pragma once

#include <atomic>
#include <mutex>

namespace saf {

class SmemLimit {
 public:
  // Calls set(bytes) (0: done) unless the limit of device `dev` is there
  // already, and returns what it returned.  Calls to set never overlap and
  // never lower a limit: between two threads that both found it too low, the
  // smaller request could otherwise land last and the larger be remembered.
  template <class Set>
  int raise(int dev, int bytes, Set set) {
    const bool known = dev >= 0 && dev < kDevices;
    if (known && at_[dev].load(std::memory_order_acquire) >= bytes) return 0;
    const std::lock_guard<std::mutex> lock(mutex_);
    if (known && at_[dev].load(std::memory_order_relaxed) >= bytes) return 0;
    const int rc = set(bytes);
    if (rc == 0 && known) at_[dev].store(bytes, std::memory_order_release);
    return rc;
  }

 private:
  static constexpr int kDevices = 64;
  std::atomic<int> at_[kDevices] = {};
  std::mutex mutex_;
};

}  // namespace saf
