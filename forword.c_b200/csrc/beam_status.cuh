// beam_status.cuh — the error word of the beam-search kernels.
#pragma once
#include <cuda_runtime.h>

#include <cstdint>
#include <mutex>

namespace fwb {

// Set when a bounded wait of the attention kernel ran out; stays until taken.
__device__ uint32_t g_beam_err;

__global__ void beam_status_kernel(uint32_t *out) { *out = atomicExch(&g_beam_err, 0u); }

// The error word after the work queued on `st`, cleared in the same step: what
// another stream's kernel sets afterwards is the next look's.  Waits.
inline cudaError_t beam_take_status(cudaStream_t st, uint32_t &word) {
    static std::mutex one;  // look at a time: they share the place that the kernel writes
    static uint32_t *place = nullptr;
    const std::lock_guard<std::mutex> lock(one);
    cudaError_t e = place ? cudaSuccess : cudaHostAlloc(&place, sizeof *place, cudaHostAllocPortable);
    if (e != cudaSuccess) return e;
    beam_status_kernel<<<1, 1, 0, st>>>(place);
    e = cudaGetLastError();
    if (e == cudaSuccess) e = cudaStreamSynchronize(st);
    if (e == cudaSuccess) word = *static_cast<volatile uint32_t *>(place);
    return e;
}

}  // namespace fwb
