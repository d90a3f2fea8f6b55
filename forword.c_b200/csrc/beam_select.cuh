// beam_select.cuh — the selection of a beam step.
//
// For a group of n_beam rows of logits x with accumulated scores c:
//
//     score[w][v] = c[w] + (x[w][v] - lse[w]),  lse[w] = log sum_v exp(x[w][v])
//
// and the n_select largest of the group's n_beam * n_vocab scores, in
// descending order, the lower flat index w * n_vocab + v first among equals.
// A row whose lse is not finite (every token barred, or a NaN or +inf among
// its logits) or whose accumulated score is not finite offers no candidate:
// its scores are -inf.
//
// The logits are read once.  Within a row the scores order as the logits do,
// so a chunk's candidates need no lse: a first kernel takes each row in
// chunks that one block holds in registers, writes the chunk's maximum and
// sum of exponentials and every logit that can be among the row's best; a
// second kernel (one block per group) joins the sums, scores the candidates
// and ranks them.  Scores rank in 64 bits, so that logits of one row never
// tie by rounding.
#pragma once
#include "beam_attn.cuh"

namespace fwb {

constexpr int kBsThreads = 256;       // of a chunk's block
constexpr int kBsJoinThreads = 512;
constexpr uint32_t kBsMaxSelect = 128, kBsMaxBeams = 64;
constexpr uint32_t kBsPool = 1024;    // candidates that the second kernel ranks

struct BeamSelectArgs {
    const void *logits;     // [n_group * n_beam] rows, row_stride elements apart
    const float *scores;    // [n_group * n_beam]
    float *out_scores;      // [n_group][n_select]
    int32_t *parent, *token;
    uint64_t row_stride;
    uint32_t n_group, n_beam, n_vocab, n_select;
    // workspace: per chunk (row-major [row][chunk]) its candidates (logit,
    // token), their number, and (maximum, sum of exp(x - maximum))
    float2 *cand;
    uint32_t *count;
    float2 *stat;
    uint32_t n_chunk, chunk, cap;
};

// Orders like the float, as an unsigned integer (NaN is not passed).
__device__ __forceinline__ uint32_t beam_order(float v) {
    const uint32_t b = __float_as_uint(v);
    return b & 0x80000000u ? ~b : b | 0x80000000u;
}
constexpr uint32_t kBsNone = 0x007fffffu;  // beam_order(-inf): entries at or below it are no candidates

// A value t such that at least `want` of the block's N values in `vals`
// (beam_order of each thread's best) are >= t, and few more; kBsNone + 1 if
// not as many are above kBsNone.  One warp; bisection that stops at up to
// want / 2 + 8 too many.
template <int N>
__device__ __forceinline__ uint32_t beam_threshold(const uint32_t *vals, uint32_t want) {
    const uint32_t lane = threadIdx.x & 31;
    uint32_t v[N / 32], top = 0;
#pragma unroll
    for (int i = 0; i < N / 32; ++i) {
        v[i] = vals[32 * i + lane];
        top = max(top, v[i]);
    }
    top = __reduce_max_sync(0xffffffffu, top);
    uint32_t lo = kBsNone + 1, hi = top;  // count(lo) >= want, or all there is
    while (lo < hi) {
        const uint32_t mid = lo + (hi - lo + 1) / 2;
        uint32_t n = 0;
#pragma unroll
        for (int i = 0; i < N / 32; ++i) n += v[i] >= mid;
        n = __reduce_add_sync(0xffffffffu, n);
        if (n >= want) {
            lo = mid;
            if (n <= want + want / 2 + 8) break;
        } else {
            hi = mid - 1;
        }
    }
    return lo;
}

template <typename T, int E, bool VEC>
__device__ __forceinline__ void beam_load_chunk(const T *x, uint32_t n, float *v) {
    constexpr int PV = VEC ? 16 / (int)sizeof(T) : 1;  // elements per load
#pragma unroll
    for (int i = 0; i < E / PV; ++i) {
        const uint32_t at = (i * kBsThreads + threadIdx.x) * PV;
        if constexpr (VEC) {
            uint4 raw = make_uint4(0, 0, 0, 0);
            if (at + PV <= n) raw = __ldcs(reinterpret_cast<const uint4 *>(x + at));
            else if (at < n) {
                T *part = reinterpret_cast<T *>(&raw);
                for (int e = 0; e < PV; ++e)
                    if (at + e < n) part[e] = x[at + e];
            }
            const T *e16 = reinterpret_cast<const T *>(&raw);
#pragma unroll
            for (int e = 0; e < PV; ++e) v[i * PV + e] = at + e < n ? beam_to_f32(e16[e]) : -INFINITY;
        } else {
            v[i] = at < n ? beam_to_f32(x[at]) : -INFINITY;
        }
    }
}

// One chunk of a row per block, E logits per thread.
template <typename T, int E, bool VEC>
__global__ void __launch_bounds__(kBsThreads) beam_select_chunk_kernel(BeamSelectArgs a) {
    constexpr int NW = kBsThreads / 32, PV = VEC ? 16 / (int)sizeof(T) : 1;
    __shared__ float s_max[NW], s_sum[NW];
    __shared__ uint32_t s_best[kBsThreads], s_thr, s_n;
    __shared__ uint64_t s_key[NW];
    const uint32_t lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const uint32_t row = blockIdx.x / a.n_chunk, ck = blockIdx.x % a.n_chunk;
    const uint32_t v0 = ck * a.chunk, n = min(a.chunk, a.n_vocab - v0);
    const T *x = static_cast<const T *>(a.logits) + row * a.row_stride + v0;
    float v[E];
    beam_load_chunk<T, E, VEC>(x, n, v);
    float m = -INFINITY;
#pragma unroll
    for (int e = 0; e < E; ++e) m = fmaxf(m, v[e]);
    s_best[threadIdx.x] = m == -INFINITY ? kBsNone : beam_order(m);
    if (threadIdx.x == 0) s_n = 0;
    float bm = m;
#pragma unroll
    for (int o = 16; o; o >>= 1) bm = fmaxf(bm, __shfl_xor_sync(0xffffffffu, bm, o));
    if (lane == 0) s_max[warp] = bm;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < NW; ++w) bm = fmaxf(bm, s_max[w]);
    const float base = bm == -INFINITY ? 0.f : bm;
    if (warp == 0) {
        const uint32_t thr = beam_threshold<kBsThreads>(s_best, a.n_select);
        if (lane == 0) s_thr = thr;
    }
    float sum = 0.f;  // a NaN or +inf among the logits makes it NaN
#pragma unroll
    for (int e = 0; e < E; ++e) sum += exp2_fast((v[e] - base) * 1.4426950408889634f);
#pragma unroll
    for (int o = 16; o; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
    if (lane == 0) s_sum[warp] = sum;
    __syncthreads();
    const uint32_t thr = s_thr;
    const size_t list = blockIdx.x;
    float2 *cand = a.cand + list * a.cap;
    if (beam_order(m) >= thr && m > -INFINITY) {
#pragma unroll
        for (int e = 0; e < E; ++e)
            if (v[e] > -INFINITY && beam_order(v[e]) >= thr) {
                const uint32_t at = atomicAdd(&s_n, 1);
                const uint32_t tok = v0 + ((e / PV) * kBsThreads + threadIdx.x) * PV + e % PV;
                if (at < a.cap) cand[at] = make_float2(v[e], __uint_as_float(tok));
            }
    }
    __syncthreads();
    uint32_t cnt = s_n;
    if (cnt > a.cap) {  // many equal logits, or the best in few threads: exactly n_select, one after the other
        uint64_t last = ~0ull;
        for (cnt = 0; cnt < a.n_select; ++cnt) {
            uint64_t best = 0;
#pragma unroll
            for (int e = 0; e < E; ++e)
                if (v[e] > -INFINITY) {
                    float now = v[e] + 0.f;              // (-0 ties with 0)
                    asm volatile("" : "+f"(now));        // keep the keys out of registers between rounds
                    const uint32_t tok = v0 + ((e / PV) * kBsThreads + threadIdx.x) * PV + e % PV;
                    const uint64_t key = (uint64_t)beam_order(now) << 32 | (0xffffffffu - tok);
                    if (key < last && key > best) best = key;
                }
#pragma unroll
            for (int o = 16; o; o >>= 1) {
                const uint64_t other = __shfl_xor_sync(0xffffffffu, best, o);
                best = other > best ? other : best;
            }
            if (lane == 0) s_key[warp] = best;
            __syncthreads();
#pragma unroll
            for (int w = 0; w < NW; ++w) best = s_key[w] > best ? s_key[w] : best;
            __syncthreads();
            if (threadIdx.x == 0) {
                const uint32_t u = (uint32_t)(best >> 32);
                cand[cnt] = make_float2(__uint_as_float(u & 0x80000000u ? u & 0x7fffffffu : ~u),
                                        __uint_as_float(0xffffffffu - (uint32_t)best));
            }
            last = best;
        }
    }
    if (threadIdx.x == 0) {
        float t = 0.f;
#pragma unroll
        for (int w = 0; w < NW; ++w) t += s_sum[w];
        a.stat[list] = make_float2(bm, t);
        a.count[list] = cnt;
    }
}

// One block per group: the rows' log-sums, the candidates' scores, their ranks.
__global__ void __launch_bounds__(kBsJoinThreads) beam_select_join_kernel(BeamSelectArgs a) {
    __shared__ double s_off[kBsMaxBeams];     // c - lse; NaN: a row without candidates
    __shared__ uint32_t s_best[kBsJoinThreads], s_thr, s_n;
    __shared__ double s_score[kBsPool];
    __shared__ uint32_t s_flat[kBsPool];
    __shared__ double s_kd[kBsJoinThreads / 32];
    __shared__ uint32_t s_ki[kBsJoinThreads / 32];
    constexpr uint32_t NT = kBsJoinThreads, NW = NT / 32;
    const uint32_t lane = threadIdx.x & 31, warp = threadIdx.x >> 5, g = blockIdx.x;
    const size_t list0 = (size_t)g * a.n_beam * a.n_chunk;
    const uint32_t lists = a.n_beam * a.n_chunk;
    for (uint32_t w = warp; w < a.n_beam; w += NW) {
        const float2 *st = a.stat + list0 + (size_t)w * a.n_chunk;
        float m = -INFINITY;
        for (uint32_t i = lane; i < a.n_chunk; i += 32) m = fmaxf(m, st[i].x);
#pragma unroll
        for (int o = 16; o; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
        double sum = 0;
        for (uint32_t i = lane; i < a.n_chunk; i += 32) {
            const float2 v = st[i];  // a chunk of barred tokens has sum 0 (or NaN)
            sum += v.x == -INFINITY ? (double)v.y : (double)v.y * (double)expf(v.x - m);
        }
#pragma unroll
        for (int o = 16; o; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
        if (lane == 0) {
            const float c = a.scores[g * a.n_beam + w];
            const bool live = isfinite(c) && isfinite(m) && sum > 0 && isfinite(sum);
            s_off[w] = live ? (double)c - ((double)m + log(sum)) : nan("");
        }
    }
    if (threadIdx.x == 0) s_n = 0;
    __syncthreads();
    const uint64_t slots = (uint64_t)lists * a.cap;
    auto score_of = [&](uint64_t i, double &s, uint32_t &flat) {
        const uint32_t list = (uint32_t)(i / a.cap), w = list / a.n_chunk;
        if ((uint32_t)(i % a.cap) >= a.count[list0 + list]) return false;
        const float2 c = a.cand[list0 * a.cap + i];
        s = s_off[w] + (double)c.x;
        flat = w * a.n_vocab + __float_as_uint(c.y);
        return s == s;
    };
    uint32_t best = kBsNone;
    for (uint64_t i = threadIdx.x; i < slots; i += NT) {
        double s;
        uint32_t flat;
        if (score_of(i, s, flat)) best = max(best, beam_order((float)s));
    }
    s_best[threadIdx.x] = best;
    __syncthreads();
    if (warp == 0) {
        const uint32_t thr = beam_threshold<kBsJoinThreads>(s_best, a.n_select);
        if (lane == 0) s_thr = thr;
    }
    __syncthreads();
    const uint32_t thr = s_thr;
    if (best >= thr)
        for (uint64_t i = threadIdx.x; i < slots; i += NT) {
            double s;
            uint32_t flat;
            if (score_of(i, s, flat) && beam_order((float)s) >= thr) {
                const uint32_t at = atomicAdd(&s_n, 1);
                if (at < kBsPool) {
                    s_score[at] = s;
                    s_flat[at] = flat;
                }
            }
        }
    __syncthreads();
    uint32_t n = s_n;
    __syncthreads();
    if (n > kBsPool) {  // the best in few threads: one after the other
        double ls = INFINITY;
        uint32_t li = 0;
        for (n = 0; n < a.n_select; ++n) {
            double bs = -INFINITY;
            uint32_t bi = 0xffffffffu;
            for (uint64_t i = threadIdx.x; i < slots; i += NT) {
                double s;
                uint32_t flat;
                if (!score_of(i, s, flat)) continue;
                if (n && !(s < ls || (s == ls && flat > li))) continue;
                if (s > bs || (s == bs && flat < bi)) { bs = s; bi = flat; }
            }
#pragma unroll
            for (int o = 16; o; o >>= 1) {
                const double os = __shfl_xor_sync(0xffffffffu, bs, o);
                const uint32_t oi = __shfl_xor_sync(0xffffffffu, bi, o);
                if (os > bs || (os == bs && oi < bi)) { bs = os; bi = oi; }
            }
            if (lane == 0) { s_kd[warp] = bs; s_ki[warp] = bi; }
            __syncthreads();
            for (uint32_t w = 0; w < NW; ++w)
                if (s_kd[w] > bs || (s_kd[w] == bs && s_ki[w] < bi)) { bs = s_kd[w]; bi = s_ki[w]; }
            if (threadIdx.x == 0) { s_score[n] = bs; s_flat[n] = bi; }
            __syncthreads();
            ls = bs;
            li = bi;
        }
    }
    const size_t out = (size_t)g * a.n_select;
    for (uint32_t i = threadIdx.x; i < n; i += NT) {
        const double s = s_score[i];
        const uint32_t flat = s_flat[i];
        uint32_t rank = 0;
        for (uint32_t j = 0; j < n; ++j) rank += s_score[j] > s || (s_score[j] == s && s_flat[j] < flat);
        if (rank < a.n_select) {
            a.out_scores[out + rank] = (float)s;
            a.parent[out + rank] = (int32_t)(flat / a.n_vocab);
            a.token[out + rank] = (int32_t)(flat % a.n_vocab);
        }
    }
    if (n < a.n_select && threadIdx.x < a.n_select) {
        // Fewer candidates than places: entries at -inf by index.  All
        // candidates are in the pool, so of the first n_select indexes those
        // outside it are enough.
        const uint32_t f = threadIdx.x;
        uint32_t below = 0;
        bool in = false;
        for (uint32_t j = 0; j < n; ++j) {
            below += s_flat[j] < f;
            in |= s_flat[j] == f;
        }
        const uint32_t place = n + f - below;
        if (!in && place < a.n_select) {
            a.out_scores[out + place] = -INFINITY;
            a.parent[out + place] = (int32_t)(f / a.n_vocab);
            a.token[out + place] = (int32_t)(f % a.n_vocab);
        }
    }
}

}  // namespace fwb
