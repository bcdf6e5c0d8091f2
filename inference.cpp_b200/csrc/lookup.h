// A value that is looked up once and kept only when it was found: a lookup that failed is tried
// again by the next call.  Concurrent first calls may look it up twice.
#pragma once
#include <atomic>

namespace ib {

template <typename T>
struct Lookup {
    std::atomic<T> found{nullptr};
    template <typename F>
    T get(F f) {
        T x = found.load(std::memory_order_acquire);
        if (!x && (x = f())) found.store(x, std::memory_order_release);
        return x;
    }
};

}  // namespace ib
