// A kernel's shared-memory limit is the same for every launch: raised once per device (a second thread may do it again).
#pragma once
#include <atomic>
#include <cstdint>
#include <cuda_runtime.h>

namespace nep {

template <typename Kernel>
cudaError_t raise_shared_limit(Kernel* fn, int bytes, std::atomic<uint64_t>& raised) {
    int device = 0;
    cudaError_t e = cudaGetDevice(&device);
    if (e != cudaSuccess) return e;
    const uint64_t bit = device < 64 ? uint64_t(1) << device : 0;
    if ((raised.load(std::memory_order_acquire) & bit) != 0) return cudaSuccess;
    e = cudaFuncSetAttribute(fn, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);
    if (e == cudaSuccess) raised.fetch_or(bit, std::memory_order_release);
    return e;
}

}  // namespace nep
