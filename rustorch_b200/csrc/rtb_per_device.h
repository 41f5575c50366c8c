// Numbers that are asked of a device once and kept for the process.
#pragma once
#include <atomic>

namespace rtb {

// `kSlots` numbers above 0 for each device.  An answer of 0 (the question failed)
// is given back but not kept; nor is anything for devices beyond kDevices.
template <int kSlots>
class PerDevice {
 public:
  template <typename Ask>
  int get(int device, int slot, const Ask& ask) {
    if (device < 0 || device >= kDevices) return ask();
    std::atomic<int>& known = known_[device][slot];
    int n = known.load(std::memory_order_relaxed);
    if (n == 0) {
      n = ask();
      known.store(n, std::memory_order_relaxed);
    }
    return n;
  }

 private:
  static constexpr int kDevices = 64;
  std::atomic<int> known_[kDevices][kSlots] = {};
};

}  // namespace rtb
