// A number that the driver is asked for once per device and call site.  Plain C++, so that it can be run on the CPU.
#pragma once

#include <atomic>

namespace mvb {

class PerDevice {
 public:
  // What `ask` gives for this device, kept from the first time that it is above zero; `otherwise` where it is not.
  template <typename Ask>
  int get(int device, Ask ask, int otherwise) {
    const bool kept = device >= 0 && device < kDevices;
    if (kept) {
      const int n = known_[device].load(std::memory_order_relaxed);
      if (n > 0) return n;
    }
    const int n = ask();
    if (n <= 0) return otherwise;
    if (kept) known_[device].store(n, std::memory_order_relaxed);
    return n;
  }

 private:
  static constexpr int kDevices = 64;
  std::atomic<int> known_[kDevices] = {};
};

}  // namespace mvb
