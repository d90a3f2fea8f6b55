// beam_attn.cuh — attention of sequences that share a prefix (beam search,
// several samples of one prompt, drafted continuations).
//
// Sequence s = group * n_beam + beam.  Its keys and values are the group's
// prefix rows, held once for all its beams, followed by the sequence's own
// suffix rows; with a slot table, suffix position t of s is row t of the
// sequence group * n_beam + slots[s][t] (the ancestor that computed it; an
// entry outside 0..n_beam-1 counts as the sequence's own beam).
// Query token t of n_query sees the whole prefix and the first
// suffix_len - (n_query - 1 - t) suffix positions:
//
//     out = sum_j exp(x_j - lse) v_j,  x_j = scale q . k_j,  lse = log sum_j exp(x_j)
//
// with no visible position: out = 0, lse = -inf.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "common.cuh"

namespace fwb {

struct BeamAttnArgs {
    const void *q, *pk, *pv, *sk, *sv;
    void *out;
    float *lse;                                 // or null
    const int32_t *plen, *slen, *slots;         // or null
    size_t q_seq, q_tok, q_head;                // strides in elements
    size_t p_group, p_head, p_pos;
    size_t s_seq, s_head, s_pos;
    size_t slot_seq;
    uint32_t n_group, n_beam, n_query, n_head, n_kv, gq, hd;
    uint32_t pcap, scap;
    float scale;
};

__device__ __forceinline__ float beam_to_f32(float v) { return v; }
__device__ __forceinline__ float beam_to_f32(__half v) { return __half2float(v); }
__device__ __forceinline__ float beam_to_f32(__nv_bfloat16 v) { return __bfloat162float(v); }
template <typename T> __device__ __forceinline__ T beam_from_f32(float v);
template <> __device__ __forceinline__ float beam_from_f32<float>(float v) { return v; }
template <> __device__ __forceinline__ __half beam_from_f32<__half>(float v) { return __float2half_rn(v); }
template <> __device__ __forceinline__ __nv_bfloat16 beam_from_f32<__nv_bfloat16>(float v) {
    return __float2bfloat16_rn(v);
}

// A length read from the device, held to the positions that the cache has.
__device__ __forceinline__ uint32_t beam_len(const int32_t *len, uint32_t i, uint32_t cap) {
    if (!len) return cap;
    const int32_t n = len[i];
    return n < 0 ? 0u : min((uint32_t)n, cap);
}

constexpr int kBaThreads = 128;

// One block per (query token, query head): its warps take the positions in
// turn, each with its own running maximum, sum and weighted values.
template <typename T>
__global__ void __launch_bounds__(kBaThreads) beam_attn_rows_kernel(BeamAttnArgs a) {
    constexpr int NW = kBaThreads / 32;
    __shared__ float part[NW][128], pm[NW], pl[NW];
    const uint32_t lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const uint32_t row = blockIdx.x, h = blockIdx.y, kvh = h / a.gq;
    const uint32_t s = row / a.n_query, t = row % a.n_query, grp = s / a.n_beam;
    const T *q = static_cast<const T *>(a.q) + s * a.q_seq + t * a.q_tok + h * a.q_head;
    const T *pk = static_cast<const T *>(a.pk) + grp * a.p_group + kvh * a.p_head;
    const T *pv = static_cast<const T *>(a.pv) + grp * a.p_group + kvh * a.p_head;
    const uint32_t np = beam_len(a.plen, grp, a.pcap), ns = beam_len(a.slen, s, a.scap);
    const uint32_t hidden = a.n_query - 1 - t;
    const uint32_t n = np + (ns > hidden ? ns - hidden : 0);
    float qv[4], o[4] = {0.f, 0.f, 0.f, 0.f}, m = -INFINITY, l = 0.f;
#pragma unroll
    for (int i = 0; i < 4; ++i) qv[i] = lane + 32 * i < a.hd ? beam_to_f32(q[lane + 32 * i]) : 0.f;
    for (uint32_t j = warp; j < n; j += NW) {
        const T *k, *v;
        if (j < np) {
            k = pk + j * a.p_pos;
            v = pv + j * a.p_pos;
        } else {
            const uint32_t at = j - np;
            uint32_t b = s % a.n_beam;
            if (a.slots) {
                const uint32_t from = (uint32_t)a.slots[s * a.slot_seq + at];
                if (from < a.n_beam) b = from;
            }
            const size_t off = (size_t)(grp * a.n_beam + b) * a.s_seq + kvh * a.s_head + at * a.s_pos;
            k = static_cast<const T *>(a.sk) + off;
            v = static_cast<const T *>(a.sv) + off;
        }
        float x = 0.f;
#pragma unroll
        for (int i = 0; i < 4; ++i)
            if (lane + 32 * i < a.hd) x = fmaf(qv[i], beam_to_f32(k[lane + 32 * i]), x);
#pragma unroll
        for (int w = 16; w; w >>= 1) x += __shfl_xor_sync(0xffffffffu, x, w);
        x *= a.scale;
        const float mn = fmaxf(m, x);
        const float al = m == -INFINITY ? 0.f : expf(m - mn), e = x == -INFINITY ? 0.f : expf(x - mn);
        l = fmaf(l, al, e);
#pragma unroll
        for (int i = 0; i < 4; ++i)
            if (lane + 32 * i < a.hd) o[i] = fmaf(e, beam_to_f32(v[lane + 32 * i]), o[i] * al);
        m = mn;
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) part[warp][lane + 32 * i] = o[i];
    if (lane == 0) { pm[warp] = m; pl[warp] = l; }
    __syncthreads();
    float M = -INFINITY, L = 0.f;
    for (int w = 0; w < NW; ++w) M = fmaxf(M, pm[w]);
    for (int w = 0; w < NW; ++w) L += pm[w] == -INFINITY ? 0.f : pl[w] * expf(pm[w] - M);
    const size_t at = (size_t)row * a.n_head + h;
    for (uint32_t d = threadIdx.x; d < a.hd; d += kBaThreads) {
        float v = 0.f;
        for (int w = 0; w < NW; ++w) v += pm[w] == -INFINITY ? 0.f : part[w][d] * expf(pm[w] - M);
        static_cast<T *>(a.out)[at * a.hd + d] = beam_from_f32<T>(L > 0.f ? v / L : 0.f);
    }
    if (a.lse && threadIdx.x == 0) a.lse[at] = L > 0.f ? M + logf(L) : -INFINITY;
}

}  // namespace fwb
