// func_attr.cuh -- a kernel's right to more than 48 KB of dynamic shared
// memory.  The attribute belongs to the device that is current when it is set,
// and a process may launch on several.
#pragma once

#include <cuda_runtime.h>

#include <atomic>
#include <cstdint>

namespace dance
{

// The devices on which a kernel has it; one for each kernel.
struct SmemAllowed
{
    std::atomic<uint64_t> devices{0};

    // Sets the attribute on the current device unless it is known to be set there; a failure is not remembered.
    cudaError_t on_current(const void *kernel, int bytes)
    {
        int dev = 0;
        if (cudaError_t e = cudaGetDevice(&dev))
            return e;
        const uint64_t bit = dev < 64 ? 1ull << dev : 0ull;
        if (devices.load(std::memory_order_relaxed) & bit)
            return cudaSuccess;
        const cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);
        if (e == cudaSuccess)
            devices.fetch_or(bit, std::memory_order_relaxed);
        return e;
    }
};

} // namespace dance
