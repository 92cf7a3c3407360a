// Host work done once for each device (kernel attributes, occupancies): what it
// writes is seen by every thread that run() then lets past.  Host code only.
#pragma once

#include <atomic>
#include <mutex>

namespace b200host {

struct OncePerDevice {
  static constexpr int kDevices = 64;

  // f() until it returns 0 for `device`; its status, or 0 when it was done before.
  // `device` is below kDevices.
  template <class F>
  int run(int device, F&& f) {
    if (done[device].load(std::memory_order_acquire)) return 0;
    std::lock_guard<std::mutex> lock(mutex);
    if (done[device].load(std::memory_order_relaxed)) return 0;
    const int status = f();
    if (status == 0) done[device].store(true, std::memory_order_release);
    return status;
  }

  std::mutex mutex;
  std::atomic<bool> done[kDevices] = {};
};

}  // namespace b200host
