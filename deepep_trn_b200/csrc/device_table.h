// Answers of a device that are asked for once: one value above zero for each device and key.
#pragma once

#include <atomic>

namespace b200ep {

template <int KEYS>
class DeviceTable {
 public:
  // `ask()` gives the value of `device` (the current one); what it throws leaves the place empty. Devices past
  // the table are asked every time.
  template <typename Ask>
  int get(int device, int key, Ask ask) {
    if (device < 0 || device >= kDevices || key < 0 || key >= KEYS) return ask();
    int v = at_[device][key].load(std::memory_order_relaxed);
    if (v == 0) {
      v = ask();
      at_[device][key].store(v, std::memory_order_relaxed);
    }
    return v;
  }

 private:
  static constexpr int kDevices = 64;
  std::atomic<int> at_[kDevices][KEYS] = {};
};

}  // namespace b200ep
