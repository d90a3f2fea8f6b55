// launch.h — what the C entry points of the operators share: error texts,
// launches and device properties.
#pragma once
#include <cuda_runtime.h>

#include <cstdint>
#include <cstdio>

#include "status.h"

namespace fwb {

inline bool fail(const char *text) {
    set_last_error(text);
    return false;
}

inline bool launched(cudaError_t e, const char *who) {
    if (e == cudaSuccess) return true;
    char b[160];
    snprintf(b, sizeof b, "%s: %s", who, cudaGetErrorString(e));
    return fail(b);
}

// A kernel whose blocks may be placed while the stream's kernel before it
// ends (it waits for that one's results itself).
template <typename F, typename... A>
cudaError_t launch_after(F *fn, dim3 grid, unsigned threads, unsigned smem, unsigned cluster, cudaStream_t st, const A &...args) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = grid;
    cfg.blockDim = dim3(threads);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = st;
    cudaLaunchAttribute at[2];
    at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    at[0].val.programmaticStreamSerializationAllowed = 1;
    at[1].id = cudaLaunchAttributeClusterDimension;
    at[1].val.clusterDim.x = cluster;
    at[1].val.clusterDim.y = at[1].val.clusterDim.z = 1;
    cfg.attrs = at;
    cfg.numAttrs = cluster > 1 ? 2 : 1;
    return cudaLaunchKernelEx(&cfg, fn, args...);
}

// Dynamic shared memory past the default limit, once per kernel and device.
template <typename F>
bool opt_in(F *fn, uint32_t smem, bool (&ready)[64], const char *who) {
    int dev = 0;
    if (!launched(cudaGetDevice(&dev), who)) return false;
    if (dev < 64 && ready[dev]) return true;
    if (!launched(cudaFuncSetAttribute(fn, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem), who)) return false;
    if (dev < 64) ready[dev] = true;
    return true;
}

// Bytes of an element of GGML type F32, F16 or BF16; 0 for others.
inline uint32_t elem_bytes(uint32_t type) { return type == 0 ? 4u : type == 1 || type == 30 ? 2u : 0u; }

inline uint32_t device_sms() {
    static int n[64] = {};
    int dev = 0;
    if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) return 148;
    if (!n[dev]) {
        int v = 0;
        if (cudaDeviceGetAttribute(&v, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess || v < 1) return 148;
        n[dev] = v;
    }
    return (uint32_t)n[dev];
}

}  // namespace fwb
