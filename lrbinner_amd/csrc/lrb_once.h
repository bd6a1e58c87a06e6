// lrb_once.h -- what is done once for each device of a process (plain C++).
#ifndef LRB_ONCE_H
#define LRB_ONCE_H

#include <atomic>

// hipFuncSetAttribute is per DEVICE: a launch site remembers which devices it has raised its kernel's limit on (the C ABI allows
// contexts on several GPUs in one process).  A device counts as done behind the call and if it succeeded (0): a thread that finds
// it done may launch.  Two threads that come together both make the call.
struct lrb_per_device_once {
    std::atomic<bool> done[64] = {};
    template <typename F> auto once(int dev, F call) -> decltype(call())
    {
        const bool known = dev >= 0 && dev < 64;
        if (known && done[dev].load(std::memory_order_acquire)) return decltype(call())(0);
        const auto err = call();
        if (known && err == decltype(call())(0)) done[dev].store(true, std::memory_order_release);
        return err;
    }
};

#endif
