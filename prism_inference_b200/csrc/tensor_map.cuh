// tensor_map.cuh - the driver's tensor map encoder, resolved at run time (nothing links libcuda).
#pragma once
#include <cudaTypedefs.h>
#include <cuda_runtime.h>

#include <atomic>

namespace prism {

// NULL where the driver does not have it; asked again by the next call then
inline PFN_cuTensorMapEncodeTiled_v12000 encode_tiled() {
    static std::atomic<void*> known{nullptr};
    void* p = known.load(std::memory_order_relaxed);
    if (!p) {
        cudaDriverEntryPointQueryResult q;
        if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &p, cudaEnableDefault, &q) != cudaSuccess ||
            q != cudaDriverEntryPointSuccess)
            p = nullptr;
        known.store(p, std::memory_order_relaxed);
    }
    return reinterpret_cast<PFN_cuTensorMapEncodeTiled_v12000>(p);
}

}  // namespace prism
