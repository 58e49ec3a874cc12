// How much dynamic LDS a kernel has been allowed, per device; host code only.
#pragma once
#include <atomic>
#include <cstddef>
#include <mutex>

// A kernel that wants more than 64 KB of dynamic LDS must be told so once per device: the attribute
// belongs to the current device's copy of the kernel, so the "already done" note is kept per device
// (one static LdsLimit per kernel).  Some kernels' size varies by call: the attribute is set under a lock and only ever
// raised, so that no call lowers it between another's setting and its launch.
struct LdsLimit {
    static constexpr int MAX_DEV = 64;
    std::atomic<size_t> bytes[MAX_DEV];
    std::mutex lock;
    LdsLimit() { for (auto& b : bytes) b.store(0, std::memory_order_relaxed); }

    // set(bytes) -> true where the attribute was set; the answer is set's, or true where the limit is high enough already
    template <typename Set>
    bool raise(int device, size_t want, Set set) {
        const bool slot = device >= 0 && device < MAX_DEV;
        if (slot && bytes[device].load(std::memory_order_acquire) >= want) return true;
        std::lock_guard<std::mutex> guard(lock);
        if (slot && bytes[device].load(std::memory_order_relaxed) >= want) return true;
        if (!set(want)) return false;
        if (slot) bytes[device].store(want, std::memory_order_release);
        return true;
    }
};
