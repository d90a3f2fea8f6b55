// beam_select.cuh — the selection of a beam step.
//
// For a group of n_beam rows of logits x with accumulated scores c:
//
//     score[w][v] = c[w] + (x[w][v] - lse[w]),  lse[w] = log sum_v exp(x[w][v])
//
// and the n_select largest of the group's n_beam * n_vocab scores, in
// descending order, the lower flat index w * n_vocab + v first among equals.
// A row whose lse is not finite (every token barred, or a NaN or +inf among
// its logits) or whose accumulated score is NaN, -inf or +inf offers no
// candidate: its scores are -inf.
#pragma once
#include "beam_attn.cuh"

namespace fwb {

struct BeamSelectArgs {
    const void *logits;     // [n_group * n_beam] rows, row_stride elements apart
    const float *scores;    // [n_group * n_beam]
    float *out_scores;      // [n_group][n_select]
    int32_t *parent, *token;
    uint64_t *cand;         // workspace
    float *stat;
    uint64_t row_stride;
    uint32_t n_group, n_beam, n_vocab, n_select;
};

// Orders like the float, as an unsigned integer; NaN is not passed.
__device__ __forceinline__ uint32_t beam_order(float v) {
    const uint32_t b = __float_as_uint(v + 0.f);  // -0 -> +0: equal scores compare equal
    return b & 0x80000000u ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ float beam_unorder(uint32_t u) {
    return __uint_as_float(u & 0x80000000u ? u & 0x7fffffffu : ~u);
}

constexpr int kBsThreads = 512;

// The score of one entry: the row's own roundings in this order.
__device__ __forceinline__ float beam_score(float x, float top, float logsum, float c, bool live) {
    return live ? __fadd_rn(__fsub_rn(__fsub_rn(x, top), logsum), c) : -INFINITY;
}

// One block per group: the rows' log-sums, then one pass over the group for
// each selected entry.
template <typename T>
__global__ void __launch_bounds__(kBsThreads) beam_select_passes_kernel(BeamSelectArgs a) {
    __shared__ float s_top[64], s_log[64], s_red[kBsThreads / 32];
    __shared__ uint64_t s_key[kBsThreads / 32], s_best;
    __shared__ uint32_t s_live[64];
    const uint32_t lane = threadIdx.x & 31, warp = threadIdx.x >> 5, g = blockIdx.x;
    constexpr uint32_t NW = kBsThreads / 32;
    for (uint32_t w = 0; w < a.n_beam; ++w) {
        const T *x = static_cast<const T *>(a.logits) + (size_t)(g * a.n_beam + w) * a.row_stride;
        float m = -INFINITY, nan = 0.f;
        for (uint32_t v = threadIdx.x; v < a.n_vocab; v += kBsThreads) {
            const float f = beam_to_f32(x[v]);
            m = fmaxf(m, f);
            if (f != f) nan = 1.f;
        }
        for (int o = 16; o; o >>= 1) {
            m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
            nan = fmaxf(nan, __shfl_xor_sync(0xffffffffu, nan, o));
        }
        if (nan != 0.f) m = INFINITY;
        if (lane == 0) s_red[warp] = m;
        __syncthreads();
        for (uint32_t i = 0; i < NW; ++i) m = fmaxf(m, s_red[i]);
        __syncthreads();
        float sum = 0.f;
        if (m > -INFINITY && m < INFINITY)
            for (uint32_t v = threadIdx.x; v < a.n_vocab; v += kBsThreads) sum += expf(beam_to_f32(x[v]) - m);
        for (int o = 16; o; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
        if (lane == 0) s_red[warp] = sum;
        __syncthreads();
        sum = 0.f;
        for (uint32_t i = 0; i < NW; ++i) sum += s_red[i];
        const float c = a.scores[g * a.n_beam + w];
        if (threadIdx.x == 0) {
            s_top[w] = m;
            s_log[w] = logf(sum);
            s_live[w] = m > -INFINITY && m < INFINITY && isfinite(c);
        }
        __syncthreads();
    }
    uint64_t last = ~0ull;
    for (uint32_t k = 0; k < a.n_select; ++k) {  // the largest key below the last one taken
        uint64_t best = 0;
        for (uint32_t w = 0; w < a.n_beam; ++w) {
            const T *x = static_cast<const T *>(a.logits) + (size_t)(g * a.n_beam + w) * a.row_stride;
            const float c = a.scores[g * a.n_beam + w];
            for (uint32_t v = threadIdx.x; v < a.n_vocab; v += kBsThreads) {
                const float sc = beam_score(beam_to_f32(x[v]), s_top[w], s_log[w], c, s_live[w]);
                const uint64_t key = (uint64_t)beam_order(sc) << 32 | (0xffffffffu - (w * a.n_vocab + v));
                if (key < last && key > best) best = key;
            }
        }
        for (int o = 16; o; o >>= 1) {
            const uint64_t other = __shfl_xor_sync(0xffffffffu, best, o);
            best = other > best ? other : best;
        }
        if (lane == 0) s_key[warp] = best;
        __syncthreads();
        if (threadIdx.x == 0) {
            for (uint32_t i = 0; i < NW; ++i) best = s_key[i] > best ? s_key[i] : best;
            s_best = best;
            const uint32_t flat = 0xffffffffu - (uint32_t)best;
            const size_t at = (size_t)g * a.n_select + k;
            a.out_scores[at] = beam_unorder((uint32_t)(best >> 32));
            a.parent[at] = (int32_t)(flat / a.n_vocab);
            a.token[at] = (int32_t)(flat % a.n_vocab);
        }
        __syncthreads();
        last = s_best;
        __syncthreads();
    }
}

}  // namespace fwb
