// A number that a device is asked for once, kept apart for each device.
#pragma once

#include <atomic>

namespace esmb200 {

class PerDevice {
 public:
  // `ask` gives the number, or 0 if the device cannot say: then it is asked again
  // next time, like a device beyond the last one that has a place.
  template <typename Ask>
  int get(int device, Ask ask) {
    if (device < 0 || device >= kDevices) return ask();
    int n = known_[device].load(std::memory_order_relaxed);
    if (n == 0) {
      n = ask();
      known_[device].store(n, std::memory_order_relaxed);
    }
    return n;
  }

 private:
  static constexpr int kDevices = 64;
  std::atomic<int> known_[kDevices] = {};
};

}  // namespace esmb200
