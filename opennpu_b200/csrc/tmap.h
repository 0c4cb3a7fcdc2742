// Host side of TMA tensor maps: the driver's encode function, looked up once.
#pragma once
#include <cuda.h>
#include <cuda_runtime.h>
#include <cudaTypedefs.h>

#include <atomic>

namespace onpu_b200 {

// Calls of several threads may be the first at once: each that finds nothing yet looks for itself, and only a function that
// was found is kept.
inline PFN_cuTensorMapEncodeTiled_v12000 tensor_map_encode_fn() {
    static std::atomic<PFN_cuTensorMapEncodeTiled_v12000> kept{nullptr};
    if (const auto fn = kept.load(std::memory_order_acquire)) return fn;
    void *ptr = nullptr;
    cudaDriverEntryPointQueryResult q{};
    if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &ptr, cudaEnableDefault, &q) != cudaSuccess ||
        q != cudaDriverEntryPointSuccess)
        return nullptr;
    const auto fn = reinterpret_cast<PFN_cuTensorMapEncodeTiled_v12000>(ptr);
    kept.store(fn, std::memory_order_release);
    return fn;
}

}  // namespace onpu_b200
