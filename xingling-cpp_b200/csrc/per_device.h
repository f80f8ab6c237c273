// A number that is asked of each device once and kept, by any thread: 0 while
// it is not known.  Shared by the library and by the check that runs on the
// host.
#pragma once
#include <atomic>

namespace xl {

class PerDevice {
public:
    static constexpr int kDevices = 64;  // further ones are asked every time
    // What is kept for the device, else ask() and, where that is positive, keep it.
    template <typename Ask>
    int get(int device, Ask ask) {
        const bool kept = device >= 0 && device < kDevices;
        int v = kept ? known_[device].load(std::memory_order_relaxed) : 0;
        if (v) return v;
        v = ask();
        if (kept && v > 0) known_[device].store(v, std::memory_order_relaxed);
        return v;
    }

private:
    std::atomic<int> known_[kDevices] = {};
};

}  // namespace xl
