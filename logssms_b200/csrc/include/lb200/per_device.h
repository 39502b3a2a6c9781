// What a launcher remembers between calls about a kernel, for each device of the process by itself: how far its limit of dynamic
// shared memory has been raised there, and what a query has answered.  Devices past the last place are asked every time.
#pragma once
#include <atomic>
#include <cstddef>

namespace lb200 {

constexpr int kRememberedDevices = 64;

struct SharedLimits {
    static constexpr size_t kDefault = 48 * 1024;         // what every kernel may have unasked
    std::atomic<size_t> have[kRememberedDevices] = {};
    // `set(bytes)` raises the limit on `device` and returns an error code; its success is remembered, its failure is not
    template <typename Set>
    int raise(int device, size_t bytes, Set set) {
        const bool known = device >= 0 && device < kRememberedDevices;
        if (bytes <= kDefault || (known && bytes <= have[device].load(std::memory_order_relaxed))) return 0;
        const int rc = set(bytes);
        if (rc == 0 && known) have[device].store(bytes, std::memory_order_relaxed);
        return rc;
    }
};

struct AskedOnce {
    std::atomic<int> answer[kRememberedDevices] = {};     // the answer + 1; 0: not asked yet
    // `ask()`: a number from 0 up
    template <typename Ask>
    int get(int device, Ask ask) {
        const bool known = device >= 0 && device < kRememberedDevices;
        const int seen = known ? answer[device].load(std::memory_order_relaxed) : 0;
        if (seen > 0) return seen - 1;
        const int n = ask();
        if (known) answer[device].store(n + 1, std::memory_order_relaxed);
        return n;
    }
};

}  // namespace lb200
