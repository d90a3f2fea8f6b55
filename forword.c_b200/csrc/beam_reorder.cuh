// beam_reorder.cuh — per-beam state moved by the parents of a beam step.
//
// State of shape [n_outer][n_group * n_beam][n_inner] runs of run_bytes bytes:
//
//     dst[o][g * n_beam + b][i] = src[o][g * n_beam + parent[g][b]][i]
//
// in place (dst == src) or into another buffer; a parent outside
// 0..n_beam-1 counts as b itself.  In place every byte column
// of a group is read for all its beams before any of it is written, by the
// one thread that owns the column, so no second buffer and no ordering
// between threads is needed.
#pragma once
#include "common.cuh"

namespace fwb {

struct BeamReorderArgs {
    const uint8_t *src;
    uint8_t *dst;
    const int32_t *parent;                                // [n_group][n_beam]
    size_t src_outer, src_slot, src_inner;                // strides in bytes
    size_t dst_outer, dst_slot, dst_inner;
    uint32_t n_group, n_beam, n_outer, n_inner, n_col;    // n_col: columns of sizeof(V) bytes in a run
};

constexpr int kBrThreads = 256;
constexpr uint32_t kBrMaxBeams = 64;

// V: the column's type (16, 4 or 1 bytes); NB: the most beams of a group.
template <typename V, int NB>
__global__ void __launch_bounds__(kBrThreads) beam_reorder_kernel(BeamReorderArgs a) {
    const uint64_t n = (uint64_t)a.n_outer * a.n_group * a.n_inner * a.n_col;
    for (uint64_t i = (uint64_t)blockIdx.x * kBrThreads + threadIdx.x; i < n; i += (uint64_t)gridDim.x * kBrThreads) {
        const uint32_t col = i % a.n_col;
        uint64_t r = i / a.n_col;
        const uint32_t in = r % a.n_inner;
        r /= a.n_inner;
        const uint32_t g = r % a.n_group, o = r / a.n_group;
        const uint8_t *src = a.src + o * a.src_outer + in * a.src_inner + (size_t)col * sizeof(V);
        uint8_t *dst = a.dst + o * a.dst_outer + in * a.dst_inner + (size_t)col * sizeof(V);
        const int32_t *par = a.parent + (size_t)g * a.n_beam;
        V v[NB];
#pragma unroll
        for (int b = 0; b < NB; ++b)
            if (b < a.n_beam) {
                const uint32_t p = (uint32_t)par[b] < a.n_beam ? (uint32_t)par[b] : (uint32_t)b;
                v[b] = *reinterpret_cast<const V *>(src + ((size_t)g * a.n_beam + p) * a.src_slot);
            }
#pragma unroll
        for (int b = 0; b < NB; ++b)
            if (b < a.n_beam) *reinterpret_cast<V *>(dst + ((size_t)g * a.n_beam + b) * a.dst_slot) = v[b];
    }
}

}  // namespace fwb
