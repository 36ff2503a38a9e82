// gk_once.h -- values that the engine looks up once per device and keeps for the process.
#pragma once

#include <atomic>

namespace gk {

// What `look_up` gives for a device, kept from the first call on; any thread may ask at any time
// (two that ask first both look up, and store the same). T{} stands for "not known yet": a look-up
// that fails gives it, and is tried again by the next call. Indices past 63 share entries.
template <typename T>
class PerDevice {
public:
    template <typename F>
    T get(int dev, F look_up) {
        std::atomic<T>& at = value_[dev & 63];
        T v = at.load(std::memory_order_acquire);
        if (v == T{}) {
            v = look_up();
            at.store(v, std::memory_order_release);
        }
        return v;
    }

private:
    std::atomic<T> value_[64] = {};
};

}  // namespace gk
