// tensor_map.h — cuTensorMapEncodeTiled from the driver (through the runtime's
// entry-point query, so the library does not link libcuda itself).
#pragma once
#include <cuda.h>
#include <cuda_runtime.h>

namespace fwb {

// null where the driver has none
inline decltype(&cuTensorMapEncodeTiled) tensor_map_encoder() {
    static const auto fn = [] {
        void *p = nullptr;
        cudaDriverEntryPointQueryResult q{};
        const bool ok = cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &p, cudaEnableDefault, &q) == cudaSuccess &&
                        q == cudaDriverEntryPointSuccess;
        return ok ? reinterpret_cast<decltype(&cuTensorMapEncodeTiled)>(p) : nullptr;
    }();
    return fn;
}

}  // namespace fwb
