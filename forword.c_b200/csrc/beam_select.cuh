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
// so the candidates of a part of a row need no lse: a first kernel streams
// parts of rows, keeping the running maximum and sum of exponentials per
// thread and the logits that can still be among the part's best; a second
// kernel (one block per group) joins the sums, scores the candidates and
// ranks them.  Scores rank in 64 bits, so that logits of one row never tie by
// rounding.
#pragma once
#include <cooperative_groups.h>

#include "beam_attn.cuh"

namespace fwb {

constexpr int kBsThreads = 256;       // of a part's block
constexpr int kBsJoinThreads = 512;
constexpr uint32_t kBsJoinCluster = 8;  // most blocks of a group's join
constexpr uint32_t kBsMaxSelect = 128, kBsMaxBeams = 64;
constexpr uint32_t kBsList = 1024;    // candidates that a block of the first kernel holds
constexpr uint32_t kBsPool = 2048;    // candidates that the second kernel ranks
constexpr int kBsLogits = 16;         // of a thread and piece

struct BeamSelectArgs {
    const void *logits;     // [n_group * n_beam] rows, row_stride elements apart
    const float *scores;    // [n_group * n_beam]
    float *out_scores;      // [n_group][n_select]
    int32_t *parent, *token;
    uint64_t row_stride;
    uint32_t n_group, n_beam, n_vocab, n_select;
    // workspace: per part (row-major [row][part]) `cap` candidates (logit,
    // token; a NaN logit in unused places) and (m, sum of exp(x - m)), m the
    // largest logit
    float2 *cand;
    float2 *stat;
    uint32_t n_part, part, cap;
};

// Orders like the float, as an unsigned integer (NaN is not passed; -0 and 0
// are equal).
__device__ __forceinline__ uint32_t beam_order(float v) {
    const uint32_t b = __float_as_uint(v + 0.f);
    return b & 0x80000000u ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ float beam_unorder(uint32_t u) {
    return __uint_as_float(u & 0x80000000u ? u & 0x7fffffffu : ~u);
}
constexpr uint32_t kBsNone = 0x007fffffu;  // beam_order(-inf): entries at or below it are no candidates

// A value t such that at least `want` of the block's N values in `vals`
// (beam_order of each thread's best) are >= t, and few more; kBsNone + 1 if
// not as many are above kBsNone.  One warp; bisection between the least and
// the largest value that stops at up to want / 2 + 8 too many.
template <int N>
__device__ __forceinline__ uint32_t beam_threshold(const uint32_t *vals, uint32_t want) {
    const uint32_t lane = threadIdx.x & 31;
    uint32_t v[N / 32], top = 0, least = 0xffffffffu, some = 0;
#pragma unroll
    for (int i = 0; i < N / 32; ++i) {
        v[i] = vals[32 * i + lane];
        top = max(top, v[i]);
        if (v[i] > kBsNone) {
            least = min(least, v[i]);
            ++some;
        }
    }
    top = __reduce_max_sync(0xffffffffu, top);
    least = __reduce_min_sync(0xffffffffu, least);
    if (__reduce_add_sync(0xffffffffu, some) < want) return kBsNone + 1;
    uint32_t lo = least, hi = top;  // count(lo) >= want
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

// A piece: E logits of each thread, loaded 16 bytes at a time (VEC) or one.  With
// VEC the pieces ahead are copied asynchronously into shared memory; every
// thread reads only what it copied itself, so that needs no barrier.  One
// piece ahead, so that five blocks fit an SM.
constexpr int kBsStages = 2;
template <typename T, bool VEC>
struct BeamPiece {
    static constexpr int E = kBsLogits, PV = VEC ? 16 / (int)sizeof(T) : 1;  // elements per load
    static constexpr uint32_t kLogits = E * kBsThreads;
    static constexpr uint32_t kSmem = VEC ? kBsStages * kLogits * sizeof(T) : 0;
    static __device__ __forceinline__ uint32_t at(int e) { return ((e / PV) * kBsThreads + threadIdx.x) * PV + e % PV; }
    // starts the copies of a piece; x: its first logit, n: logits from there on
    static __device__ __forceinline__ void start(const T *x, uint32_t n, T *stage) {
        if constexpr (VEC) {
#pragma unroll
            for (int i = 0; i < E / PV; ++i) {
                const uint32_t p = at(i * PV);
                if (p + PV <= n) cp_async16(stage + p, x + p);
            }
            cp_async_commit();
        }
    }
    // the piece's logits, -inf past n
    static __device__ __forceinline__ void load(const T *x, uint32_t n, const T *stage, float *v) {
        if constexpr (VEC) {
            cp_async_wait<1>();
#pragma unroll
            for (int i = 0; i < E / PV; ++i) {
                const uint4 raw = *reinterpret_cast<const uint4 *>(stage + at(i * PV));
#pragma unroll
                for (int e = 0; e < PV; ++e) v[i * PV + e] = beam_to_f32(reinterpret_cast<const T *>(&raw)[e]);
            }
            if (n < kLogits)
#pragma unroll
                for (int e = 0; e < E; ++e)
                    if (at(e - e % PV) + PV > n) v[e] = at(e) < n ? beam_to_f32(x[at(e)]) : -INFINITY;
        } else {
#pragma unroll
            for (int e = 0; e < E; ++e) v[e] = at(e) < n ? beam_to_f32(x[at(e)]) : -INFINITY;
        }
    }
};

// The candidates that a block has gathered so far.
struct BeamList {
    float x[kBsList];
    uint32_t tok[kBsList];
    uint32_t n, thr;
    uint32_t best[kBsThreads];
    uint64_t key[kBsThreads / 32];
};

// Raises thr to about the n_select-th best of the list and drops what is
// below; a list that equal logits keep long is cut to exactly n_select (the
// pieces come in the order of the tokens, so later equals cannot displace
// them, and thr excludes these).  The whole block.
__device__ __noinline__ void beam_trim(BeamList &l, uint32_t want) {
    constexpr uint32_t PT = kBsList / kBsThreads;
    const uint32_t n = min(l.n, kBsList);
    float x[PT], best = -INFINITY;
    uint32_t tok[PT];
#pragma unroll
    for (uint32_t i = 0; i < PT; ++i) {
        const uint32_t j = i * kBsThreads + threadIdx.x;
        x[i] = j < n ? l.x[j] : -INFINITY;
        tok[i] = j < n ? l.tok[j] : 0;
        best = fmaxf(best, x[i]);
    }
    l.best[threadIdx.x] = best == -INFINITY ? kBsNone : beam_order(best);
    __syncthreads();
    if (threadIdx.x < 32) {
        const uint32_t thr = beam_threshold<kBsThreads>(l.best, want);
        if (threadIdx.x == 0) {
            l.thr = max(l.thr, thr);
            l.n = 0;
        }
    }
    __syncthreads();
    const float thr = beam_unorder(l.thr);
#pragma unroll
    for (uint32_t i = 0; i < PT; ++i)
        if (x[i] >= thr) {
            const uint32_t at = atomicAdd(&l.n, 1);
            l.x[at] = x[i];
            l.tok[at] = tok[i];
        }
    __syncthreads();
    const uint32_t kept = l.n;
    if (kept <= kBsList / 2) return;
    uint32_t rank[PT];
#pragma unroll
    for (uint32_t i = 0; i < PT; ++i) {
        const uint32_t j = i * kBsThreads + threadIdx.x;
        rank[i] = kept;
        if (j < kept) {
            x[i] = l.x[j];
            tok[i] = l.tok[j];
            rank[i] = 0;
            for (uint32_t k = 0; k < kept; ++k)
                rank[i] += (uint32_t)(l.x[k] > x[i]) | ((uint32_t)(l.x[k] == x[i]) & (uint32_t)(l.tok[k] < tok[i]));
        }
    }
    __syncthreads();
#pragma unroll
    for (uint32_t i = 0; i < PT; ++i)
        if (rank[i] < want) {
            l.x[rank[i]] = x[i];
            l.tok[rank[i]] = tok[i];
            if (rank[i] == want - 1) {
                l.n = want;
                l.thr = max(l.thr, beam_order(x[i]) + 1);
            }
        }
    __syncthreads();
}

// The n_select best of a piece (more than that many) behind the first `old`
// entries of the list, one after the other, read from memory again.  The
// whole block.
template <typename T>
__device__ __noinline__ void beam_take_best(BeamList &l, const T *x, uint32_t n, uint32_t tok0, uint32_t old,
                                            uint32_t want) {
    constexpr uint32_t NW = kBsThreads / 32;
    uint64_t last = ~0ull;
    for (uint32_t k = 0; k < want; ++k) {
        uint64_t best = 0;
        for (uint32_t i = threadIdx.x; i < n; i += kBsThreads) {
            const float v = beam_to_f32(x[i]);
            const uint64_t key = (uint64_t)beam_order(v) << 32 | (0xffffffffu - (tok0 + i));
            if (v > -INFINITY && key < last && key > best) best = key;
        }
#pragma unroll
        for (int o = 16; o; o >>= 1) {
            const uint64_t other = __shfl_xor_sync(0xffffffffu, best, o);
            best = other > best ? other : best;
        }
        if (threadIdx.x % 32 == 0) l.key[threadIdx.x / 32] = best;
        __syncthreads();
        for (uint32_t w = 0; w < NW; ++w) best = l.key[w] > best ? l.key[w] : best;
        if (threadIdx.x == 0) {
            const uint32_t u = (uint32_t)(best >> 32);
            l.x[old + k] = beam_unorder(u);
            l.tok[old + k] = 0xffffffffu - (uint32_t)best;
            l.n = old + k + 1;
            // later pieces' equals of the last one taken cannot displace it
            if (k + 1 == want) l.thr = max(l.thr, u + 1);
        }
        last = best;
        __syncthreads();
    }
}

// A piece with more logits at or above the threshold than the list has room
// for (rising logits; equal ones): the list without this piece's, then a
// threshold from this piece, or else its n_select best, read from memory
// again.  The whole block.
template <typename T>
__device__ __noinline__ void beam_overflow(BeamList &l, const T *x, uint32_t n, uint32_t tok0, uint32_t want) {
    constexpr uint32_t PT = kBsList / kBsThreads;
    float keep[PT];
    uint32_t tok[PT];
#pragma unroll
    for (uint32_t i = 0; i < PT; ++i) {
        keep[i] = l.x[i * kBsThreads + threadIdx.x];
        tok[i] = l.tok[i * kBsThreads + threadIdx.x];
    }
    float m = -INFINITY;
    for (uint32_t i = threadIdx.x; i < n; i += kBsThreads) m = fmaxf(m, beam_to_f32(x[i]));
    l.best[threadIdx.x] = m == -INFINITY ? kBsNone : beam_order(m);
    __syncthreads();
    if (threadIdx.x < 32) {
        const uint32_t t = beam_threshold<kBsThreads>(l.best, want);
        if (threadIdx.x == 0) {
            l.thr = max(l.thr, t);
            l.n = 0;
        }
    }
    __syncthreads();
#pragma unroll
    for (uint32_t i = 0; i < PT; ++i)
        if (tok[i] < tok0) {
            const uint32_t at = atomicAdd(&l.n, 1);
            l.x[at] = keep[i];
            l.tok[at] = tok[i];
        }
    __syncthreads();
    const uint32_t old = l.n;
    const float thr = beam_unorder(l.thr);
    __syncthreads();
    for (uint32_t i = threadIdx.x; i < n; i += kBsThreads) {
        const float v = beam_to_f32(x[i]);
        if (v >= thr) {
            const uint32_t at = atomicAdd(&l.n, 1);
            if (at < kBsList) {
                l.x[at] = v;
                l.tok[at] = tok0 + i;
            }
        }
    }
    __syncthreads();
    const bool still = l.n > kBsList;
    __syncthreads();
    if (still) beam_take_best(l, x, n, tok0, old, want);
}

// Two fp32 at once: x = (x + a) * s, and x += y.
__device__ __forceinline__ void beam_scaled2(float &x0, float &x1, float a, float s) {
    asm("{\n\t.reg .b64 x, y, z;\n\tmov.b64 x, {%0, %1};\n\tmov.b64 y, {%2, %2};\n\tmov.b64 z, {%3, %3};\n\t"
        "add.rn.f32x2 x, x, y;\n\tmul.rn.f32x2 x, x, z;\n\tmov.b64 {%0, %1}, x;\n\t}"
        : "+f"(x0), "+f"(x1) : "f"(a), "f"(s));
}
__device__ __forceinline__ void beam_add2(float &x0, float &x1, float y0, float y1) {
    asm("{\n\t.reg .b64 x, y;\n\tmov.b64 x, {%0, %1};\n\tmov.b64 y, {%2, %3};\n\t"
        "add.rn.f32x2 x, x, y;\n\tmov.b64 {%0, %1}, x;\n\t}"
        : "+f"(x0), "+f"(x1) : "f"(y0), "f"(y1));
}

// One part of a row per block.
//
// Bound: the logits once from DRAM.  Five blocks per SM with one piece ahead
// each keep about 80 KB of loads in flight; a logit costs about seven
// instructions (maximum, 2^x with half of a packed addition and product and one
// MUFU, half of a packed sum, a compare per four).  256 fp32 rows of 128256: 38 us on the device with the join (3.5 TB/s); the blocks
// are 3.5 per SM on average and 4 on the busiest.
template <typename T, bool VEC>
__global__ void __launch_bounds__(kBsThreads, 5) beam_select_part_kernel(BeamSelectArgs a) {
    using Piece = BeamPiece<T, VEC>;
    constexpr int NW = kBsThreads / 32, E = Piece::E;
    constexpr uint32_t kPiece = Piece::kLogits;
    constexpr float kLog2e = 1.4426950408889634f;
    extern __shared__ __align__(16) uint8_t bs_stages[];
    T *stages = reinterpret_cast<T *>(bs_stages);
    __shared__ BeamList l;
    __shared__ float s_max[NW], s_sum[NW];
    const uint32_t lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const uint32_t row = blockIdx.x / a.n_part;
    const uint32_t v0 = blockIdx.x % a.n_part * a.part, n = min(a.part, a.n_vocab - v0);
    const T *x = static_cast<const T *>(a.logits) + row * a.row_stride + v0;
    pdl_launch();
    if (threadIdx.x == 0) l.n = 0;
    Piece::start(x, n, stages);
    uint32_t stage = 0;
    const uint32_t limit = min(kBsList / 2, 3 * a.n_select + 64);  // a longer list is trimmed, which raises the threshold
    // of this thread's logits so far: the maximum and the sum of exp(x - m), of
    // every other one apart; a NaN or +inf makes it NaN.  In the logits' own units: a maximum times
    // log2(e) would overflow at the type's lowest value, which bars tokens too.
    float m = -INFINITY, sum = 0.f, odd = 0.f, thr = 0.f;
    for (uint32_t p0 = 0; p0 < n; p0 += kPiece) {
        float v[E];
        {
            const uint32_t next = p0 + kPiece;
            Piece::start(x + next, n > next ? n - next : 0, stages + (stage ^ 1) * kPiece);
            Piece::load(x + p0, n - p0, stages + stage * kPiece, v);
            stage ^= 1;
        }
        float qm[E / 4], pm = -INFINITY;  // of four logits, of all
#pragma unroll
        for (int q = 0; q < E / 4; ++q) {
            qm[q] = fmaxf(fmaxf(v[4 * q], v[4 * q + 1]), fmaxf(v[4 * q + 2], v[4 * q + 3]));
            pm = fmaxf(pm, qm[q]);
        }
        if (p0 == 0) {  // the first threshold: about the n_select-th best of the threads' best
            l.best[threadIdx.x] = pm == -INFINITY ? kBsNone : beam_order(pm);
            __syncthreads();
            if (warp == 0) {
                const uint32_t t = beam_threshold<kBsThreads>(l.best, a.n_select);
                if (lane == 0) l.thr = t;
            }
        }
        if (pm > m) {
            if (m > -INFINITY) {  // (without a maximum so far: 0, or NaN)
                const float f = exp2_fast((m - pm) * kLog2e);
                sum *= f;
                odd *= f;
            }
            m = pm;
        }
        const float ref = m == -INFINITY ? 0.f : m;
#pragma unroll
        for (int e = 0; e < E; e += 2) {
            float x0 = v[e], x1 = v[e + 1];
            beam_scaled2(x0, x1, -ref, kLog2e);
            beam_add2(sum, odd, exp2_fast(x0), exp2_fast(x1));
        }
        if (p0 == 0) {
            __syncthreads();
            thr = beam_unorder(l.thr);  // finite: -inf and NaN are below
        }
        bool full = false;
        if (pm >= thr) {
#pragma unroll
            for (int q = 0; q < E / 4; ++q)
                if (qm[q] >= thr)
#pragma unroll
                    for (int e = 4 * q; e < 4 * q + 4; ++e)
                        if (v[e] >= thr) {
                            const uint32_t at = atomicAdd(&l.n, 1);
                            full |= at >= limit;
                            if (at < kBsList) {
                                l.x[at] = v[e];
                                l.tok[at] = v0 + p0 + Piece::at(e);
                            }
                        }
        }
        if (__syncthreads_or(full)) {
            const bool over = l.n > kBsList;
            __syncthreads();
            if (over) beam_overflow(l, x + p0, min(n - p0, kPiece), v0 + p0, a.n_select);
            if (l.n > limit) beam_trim(l, a.n_select);
            thr = beam_unorder(l.thr);
            __syncthreads();
        }
    }
    if (l.n > a.cap) beam_trim(l, a.n_select);
    float2 *cand = a.cand + (size_t)blockIdx.x * a.cap;
    const uint32_t cnt = l.n;
    if (cnt <= a.cap) {
        for (uint32_t i = threadIdx.x; i < a.cap; i += kBsThreads)
            cand[i] = i < cnt ? make_float2(l.x[i], __uint_as_float(l.tok[i])) : make_float2(NAN, 0.f);
    } else {  // many equal logits: the n_select best by rank
        for (uint32_t i = threadIdx.x; i < cnt; i += kBsThreads) {
            const float xi = l.x[i];
            const uint32_t ti = l.tok[i];
            uint32_t rank = 0;
            for (uint32_t j = 0; j < cnt; ++j)
                rank += (uint32_t)(l.x[j] > xi) | ((uint32_t)(l.x[j] == xi) & (uint32_t)(l.tok[j] < ti));
            if (rank < a.n_select) cand[rank] = make_float2(xi, __uint_as_float(ti));
        }
        for (uint32_t i = a.n_select + threadIdx.x; i < a.cap; i += kBsThreads) cand[i] = make_float2(NAN, 0.f);
    }
    float bb = m;
#pragma unroll
    for (int o = 16; o; o >>= 1) bb = fmaxf(bb, __shfl_xor_sync(0xffffffffu, bb, o));
    if (lane == 0) s_max[warp] = bb;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < NW; ++w) bb = fmaxf(bb, s_max[w]);
    // a thread without finite logits has sum 0, or NaN
    sum += odd;
    if (m > -INFINITY) sum *= exp2_fast((m - bb) * kLog2e);
#pragma unroll
    for (int o = 16; o; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
    if (lane == 0) s_sum[warp] = sum;
    __syncthreads();
    if (threadIdx.x == 0) {
        float t = 0.f;
#pragma unroll
        for (int w = 0; w < NW; ++w) t += s_sum[w];
        a.stat[blockIdx.x] = make_float2(bb, t);
    }
}

// Orders like the double, as an unsigned integer.
__device__ __forceinline__ uint64_t beam_order64(double v) {
    const uint64_t b = (uint64_t)__double_as_longlong(v + 0.0);
    return b >> 63 ? ~b : b | 1ull << 63;
}
__device__ __forceinline__ double beam_unorder64(uint64_t u) {
    return __longlong_as_double((long long)(u >> 63 ? u & ~(1ull << 63) : ~u));
}

// A cluster of blocks per group: the rows' log-sums and the scores of the
// candidates; each block gives about the n_select best of its share to the
// first block's pool, which is cut and ranked.
__global__ void __launch_bounds__(kBsJoinThreads) beam_select_join_kernel(BeamSelectArgs a) {
    namespace cg = cooperative_groups;
    const cg::cluster_group cluster = cg::this_cluster();
    constexpr float kLog2e = 1.4426950408889634f;
    // a score is (x - m) + (c - log sum exp(x - m)), m the row's largest logit: x -
    // m first, since lse itself may be too large to hold the logarithm
    __shared__ float s_top[kBsMaxBeams];      // m
    __shared__ double s_off[kBsMaxBeams];     // c - log sum
    __shared__ float s_offf[kBsMaxBeams];     // the same rounded; NaN: a row without candidates
    __shared__ uint32_t s_best[kBsJoinThreads], s_thr, s_n;
    __shared__ uint64_t s_key[kBsPool];       // beam_order64 of the score
    __shared__ uint32_t s_flat[kBsPool];
    __shared__ uint64_t s_kd[kBsJoinThreads / 32];
    __shared__ uint32_t s_ki[kBsJoinThreads / 32];
    constexpr uint32_t NT = kBsJoinThreads, NW = NT / 32;
    const uint32_t lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const uint32_t cs = cluster.num_blocks(), cr = cluster.block_rank(), g = blockIdx.x / cs;
    const size_t list0 = (size_t)g * a.n_beam * a.n_part;
    if (threadIdx.x == 0) s_n = 0;
    pdl_wait();
    for (uint32_t w = warp; w < a.n_beam; w += NW) {
        const float2 *st = a.stat + list0 + (size_t)w * a.n_part;
        const float c = a.scores[g * a.n_beam + w];
        float m = -INFINITY;
        for (uint32_t i = lane; i < a.n_part; i += 32) m = fmaxf(m, st[i].x);
#pragma unroll
        for (int o = 16; o; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
        float sum = 0.f;
        for (uint32_t i = lane; i < a.n_part; i += 32) {
            const float2 v = st[i];  // a part of barred tokens has sum 0 (or NaN)
            sum += v.x == -INFINITY ? v.y : v.y * exp2_fast((v.x - m) * kLog2e);
        }
#pragma unroll
        for (int o = 16; o; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
        if (lane == 0) {
            const bool live = isfinite(c) && isfinite(m) && sum > 0 && isfinite(sum);
            const double off = (double)c - (double)logf(sum);
            s_top[w] = m;
            s_off[w] = off;
            s_offf[w] = live ? (float)off : NAN;
        }
    }
    if (cs > 1) cluster.sync();  // the offsets, and the first block's pool counter, are there
    else __syncthreads();
    uint32_t *pool_n = cluster.map_shared_rank(&s_n, 0);
    uint64_t *pool_key = cluster.map_shared_rank(s_key, 0);
    uint32_t *pool_flat = cluster.map_shared_rank(s_flat, 0);
    // The candidates in slices of 32 places, `step` warps in turn, four slices
    // at a time.  visit(logit, row, token) is called for each place (unused
    // ones and dead rows give NaN scores).
    const uint32_t per = a.cap / 32, slices = a.n_beam * a.n_part * per;
    const uint32_t places = per * a.n_part;  // slices of a row
    const float2 *cand = a.cand + list0 * a.cap;
    auto each = [&](uint32_t first, uint32_t step, auto visit) {
        for (uint32_t s0 = first; s0 < slices; s0 += 4 * step) {
            float2 c[4];
#pragma unroll
            for (int u = 0; u < 4; ++u) c[u] = cand[(size_t)min(s0 + u * step, slices - 1) * 32 + lane];
#pragma unroll
            for (int u = 0; u < 4; ++u)
                if (s0 + u * step < slices)
                    visit(c[u].x, (s0 + u * step) / places, __float_as_uint(c[u].y));
        }
    };
    float best = -INFINITY;
    each(cr * NW + warp, cs * NW, [&](float x, uint32_t w, uint32_t) { best = fmaxf(best, (x - s_top[w]) + s_offf[w]); });
    s_best[threadIdx.x] = best == -INFINITY ? kBsNone : beam_order(best);
    __syncthreads();
    if (warp == 0) {
        const uint32_t thr = beam_threshold<kBsJoinThreads>(s_best, a.n_select);
        if (lane == 0) s_thr = thr;
    }
    // The scores compared here are rounded three times in 32 bits, the
    // difference, the offset and the sum, together by at most 2^-23 of |score| +
    // |offset|: a candidate counts as below the threshold only by more than the
    // roundings of both sides.
    float off_max = 0.f;
    for (uint32_t w = 0; w < a.n_beam; ++w) off_max = fmaxf(off_max, fabsf(s_offf[w]));
    __syncthreads();
    float thr = beam_unorder(s_thr);
    thr -= 2.4e-7f * (2.f * fabsf(thr) + off_max);  // (-FLT_MAX or -inf takes all)
    if (__any_sync(0xffffffffu, best >= thr))
        each(cr * NW + warp, cs * NW, [&](float x, uint32_t w, uint32_t tok) {
            if (!((x - s_top[w]) + s_offf[w] >= thr)) return;
            const uint32_t at = atomicAdd(pool_n, 1);
            if (at < kBsPool) {
                pool_key[at] = beam_order64(((double)x - (double)s_top[w]) + s_off[w]);
                pool_flat[at] = w * a.n_vocab + tok;
            }
        });
    if (cs > 1) cluster.sync();
    else __syncthreads();
    if (cr != 0) return;
    uint32_t n = s_n;
    __syncthreads();
    if (n > kBsPool) {  // the best in few threads, or many equal scores: one after the other
        uint64_t ls = ~0ull;
        uint32_t li = 0;
        for (n = 0; n < a.n_select; ++n) {
            uint64_t bs = 0;
            uint32_t bi = 0xffffffffu;
            each(warp, NW, [&](float x, uint32_t w, uint32_t tok) {
                const float f = (x - s_top[w]) + s_offf[w];
                if (f != f) return;
                const uint64_t s = beam_order64(((double)x - (double)s_top[w]) + s_off[w]);
                const uint32_t flat = w * a.n_vocab + tok;
                if (n && !(s < ls || (s == ls && flat > li))) return;
                if (s > bs || (s == bs && flat < bi)) { bs = s; bi = flat; }
            });
#pragma unroll
            for (int o = 16; o; o >>= 1) {
                const uint64_t os = __shfl_xor_sync(0xffffffffu, bs, o);
                const uint32_t oi = __shfl_xor_sync(0xffffffffu, bi, o);
                if (os > bs || (os == bs && oi < bi)) { bs = os; bi = oi; }
            }
            if (lane == 0) { s_kd[warp] = bs; s_ki[warp] = bi; }
            __syncthreads();
            for (uint32_t w = 0; w < NW; ++w)
                if (s_kd[w] > bs || (s_kd[w] == bs && s_ki[w] < bi)) { bs = s_kd[w]; bi = s_ki[w]; }
            if (threadIdx.x == 0) { s_key[n] = bs; s_flat[n] = bi; }
            __syncthreads();
            ls = bs;
            li = bi;
        }
    } else if (n > 2 * a.n_select + 64) {  // many blocks' shares: cut once more, on the key's upper half
        constexpr uint32_t PT = kBsPool / NT;
        uint64_t key[PT];
        uint32_t flat[PT], top = 0;
#pragma unroll
        for (uint32_t i = 0; i < PT; ++i) {
            const uint32_t j = i * NT + threadIdx.x;
            key[i] = j < n ? s_key[j] : 0;
            flat[i] = j < n ? s_flat[j] : 0;
            top = max(top, (uint32_t)(key[i] >> 32));
        }
        s_best[threadIdx.x] = top;
        if (threadIdx.x == 0) s_n = 0;
        __syncthreads();
        if (warp == 0) {
            const uint32_t t = beam_threshold<kBsJoinThreads>(s_best, a.n_select);
            if (lane == 0) s_thr = t;
        }
        __syncthreads();
#pragma unroll
        for (uint32_t i = 0; i < PT; ++i)
            if (key[i] && (uint32_t)(key[i] >> 32) >= s_thr) {
                const uint32_t at = atomicAdd(&s_n, 1);
                s_key[at] = key[i];
                s_flat[at] = flat[i];
            }
        __syncthreads();
        n = s_n;
    }
    const size_t out = (size_t)g * a.n_select;
    for (uint32_t i = threadIdx.x; i < n; i += NT) {
        const uint64_t s = s_key[i];
        const uint32_t flat = s_flat[i];
        uint32_t rank = 0;
#pragma unroll 4
        for (uint32_t j = 0; j < n; ++j) rank += (uint32_t)(s_key[j] > s) | ((uint32_t)(s_key[j] == s) & (uint32_t)(s_flat[j] < flat));
        if (rank < a.n_select) {
            const uint32_t w = flat / a.n_vocab;
            a.out_scores[out + rank] = (float)beam_unorder64(s);
            a.parent[out + rank] = (int32_t)w;
            a.token[out + rank] = (int32_t)(flat - w * a.n_vocab);
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
