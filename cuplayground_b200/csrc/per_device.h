// A positive number that depends on the device (how many of a kernel's clusters it holds at once, for instance) and is asked
// for once per device. Host threads that ask at the same time store the same value.
#pragma once
#include <atomic>

namespace aristos {

class PerDevice {
public:
    // 0: not known yet, or a device beyond the table (which is asked every time)
    int get(int device) const { return inside(device) ? value_[device].load(std::memory_order_relaxed) : 0; }
    void set(int device, int value) {
        if (inside(device)) value_[device].store(value, std::memory_order_relaxed);
    }

private:
    static constexpr int MAX_DEVICES = 64;
    static bool inside(int device) { return device >= 0 && device < MAX_DEVICES; }
    std::atomic<int> value_[MAX_DEVICES] = {};
};

}  // namespace aristos
