// The limit of a kernel's dynamic shared memory. It belongs to the kernel on a
// device and not to a call: it is set once, to the most that any call asks for,
// as a call that set its own size could lower it between another host thread's
// setting and launch.
#pragma once

#include <cuda_runtime.h>

#include <atomic>

namespace fer::host {

// Devices for which a launcher keeps what it asked the runtime once.
constexpr int kMaxDevices = 64;

// Sets the kernel's limit on the current device where `known`, the kernel's own, does not have it yet.
inline cudaError_t allow_smem(const void* kernel, int most, std::atomic<bool> (&known)[kMaxDevices]) {
    int dev = 0;
    cudaError_t e = cudaGetDevice(&dev);
    if (e != cudaSuccess) return e;
    if (dev < 0 || dev >= kMaxDevices) return cudaErrorInvalidDevice;
    if (known[dev].load(std::memory_order_relaxed)) return cudaSuccess;
    e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, most);
    if (e == cudaSuccess) known[dev].store(true, std::memory_order_relaxed);
    return e;
}

}  // namespace fer::host
