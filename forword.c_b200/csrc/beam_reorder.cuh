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

// V: the column's type; NB: the most beams of a group; I: the type that
// counts all columns.  One column per thread: a thread has the loads of all
// moved beams in flight at once, which is what the memory needs.  Slots that
// keep their own state in place are neither read nor written.
// Bound: DRAM.  K/V rows of 32 layers for 8 beams, half of them moved in place
// (183 MB read and written): 35.7 us, 5.1 TB/s, of a copy's 6.5.
template <typename V, int NB, typename I>
__global__ void __launch_bounds__(kBrThreads) beam_reorder_kernel(BeamReorderArgs a) {
    const I i = (I)blockIdx.x * kBrThreads + threadIdx.x;
    I r = i / a.n_col;
    const uint32_t col = (uint32_t)(i - r * a.n_col);
    I t = r / a.n_inner;
    const uint32_t in = (uint32_t)(r - t * a.n_inner);
    const uint32_t o = (uint32_t)(t / a.n_group), g = (uint32_t)(t - (I)o * a.n_group);
    if (o >= a.n_outer) return;
    const uint8_t *src = a.src + o * a.src_outer + in * a.src_inner + (size_t)col * sizeof(V) +
                         (size_t)g * a.n_beam * a.src_slot;
    uint8_t *dst = a.dst + o * a.dst_outer + in * a.dst_inner + (size_t)col * sizeof(V) +
                   (size_t)g * a.n_beam * a.dst_slot;
    const int32_t *par = a.parent + (size_t)g * a.n_beam;
    const bool in_place = a.src == a.dst;
    V v[NB];
    uint32_t from[NB];
#pragma unroll
    for (int b = 0; b < NB; ++b)
        if (b < a.n_beam) {
            const uint32_t p = (uint32_t)par[b];
            from[b] = p < a.n_beam ? p : (uint32_t)b;
            if (!in_place || from[b] != b) v[b] = *reinterpret_cast<const V *>(src + from[b] * a.src_slot);
        }
#pragma unroll
    for (int b = 0; b < NB; ++b)
        if (b < a.n_beam && (!in_place || from[b] != b)) *reinterpret_cast<V *>(dst + b * a.dst_slot) = v[b];
}

}  // namespace fwb
