// beam_step.cuh — the small kernels of a beam step on a model: rotary
// positions with the K/V append of every beam, and fp32 -> fp16 rows.  The
// linear layers around them are the prompt path's (prefill.cuh).
#pragma once
#include "common.cuh"

namespace fwb {

// Rows [q | k | v] of beam b, all at position `pos` (rope.c:28-53, adjacent
// pairs): q to qf, k and v to row `at` of beam b's part of a layer's suffix
// caches [beam][kv_head][cap][hd].  One block per beam.
__global__ void beam_rope_kv_kernel(const float *qkv, uint32_t pos, uint32_t at, uint32_t cap, uint32_t n_q,
                                    uint32_t n_kv, uint32_t hd, const float *rope_cos, const float *rope_sin, float *qf,
                                    float *ks, float *vs) {
    const uint32_t b = blockIdx.x, half = hd >> 1, nrow = n_q + 2 * n_kv;
    const float *r = qkv + (size_t)b * nrow;
    const size_t base = (size_t)b * n_kv * cap;  // n_kv = heads * hd
    for (uint32_t g = 2 * threadIdx.x; g < nrow; g += 2 * blockDim.x) {
        const float v0 = r[g], v1 = r[g + 1];
        const uint32_t kv = g < n_q ? 0 : g < n_q + n_kv ? g - n_q : g - n_q - n_kv, d = (g < n_q ? g : kv) % hd;
        float o0 = v0, o1 = v1;
        if (g < n_q + n_kv) {
            const float c = rope_cos[(size_t)pos * half + d / 2], s = rope_sin[(size_t)pos * half + d / 2];
            o0 = __fsub_rn(__fmul_rn(v0, c), __fmul_rn(v1, s));
            o1 = __fadd_rn(__fmul_rn(v0, s), __fmul_rn(v1, c));
        }
        float *dst = g < n_q ? qf + (size_t)b * n_q + g
                             : (g < n_q + n_kv ? ks : vs) + base + ((size_t)(kv / hd) * cap + at) * hd + d;
        dst[0] = o0;
        dst[1] = o1;
    }
}

// fp32 to fp16, n a multiple of 2.
__global__ void beam_f16_kernel(const float *x, size_t n, __half *h) {
    for (size_t i = (size_t)blockIdx.x * blockDim.x + threadIdx.x; i < n / 2; i += (size_t)gridDim.x * blockDim.x) {
        const float2 v = reinterpret_cast<const float2 *>(x)[i];
        reinterpret_cast<__half2 *>(h)[i] = __floats2half2_rn(v.x, v.y);
    }
}

}  // namespace fwb
