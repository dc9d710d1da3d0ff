// smem_limit.h -- the dynamic shared memory that a kernel has been allowed, for
// launches from several threads.
#pragma once
#include <cstddef>
#include <mutex>

namespace loom {

// raise(smem) asks the driver; it is called only when a launch needs more than the
// kernel's earlier ones on the device did, and by one thread at a time: of two that
// raise the limit together, the smaller could be set last and the larger recorded.
struct SmemLimit {
    std::mutex alone;
    size_t most[16] = {};
    template <class F> auto need(int dev, size_t smem, F raise) -> decltype(raise(smem)) {
        std::lock_guard<std::mutex> hold(alone);
        if (dev < 16 && most[dev] >= smem) return {};
        const auto e = raise(smem);
        if (e == decltype(e){} && dev < 16) most[dev] = smem;
        return e;
    }
};

}  // namespace loom
