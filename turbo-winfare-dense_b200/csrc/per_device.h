// What a process does once for every device it uses: a kernel's attributes and a device's numbers belong
// to the device that was current when they were set or read.
#pragma once
#include <cuda_runtime_api.h>

#include <atomic>
#include <cstdint>

namespace g4b {

class OncePerDevice {
public:
    // Runs set() unless it has succeeded on the current device before. Threads that meet here may both
    // run it; a device past the 64th runs it every time.
    template <class Set>
    cudaError_t operator()(Set set) {
        int dev = 0;
        cudaError_t e = cudaGetDevice(&dev);
        if (e != cudaSuccess) return e;
        const uint64_t bit = dev >= 0 && dev < 64 ? 1ull << dev : 0;
        if (done_.load(std::memory_order_acquire) & bit) return cudaSuccess;
        if ((e = set()) == cudaSuccess) done_.fetch_or(bit, std::memory_order_release);
        return e;
    }

private:
    std::atomic<uint64_t> done_{0};
};

}  // namespace g4b
