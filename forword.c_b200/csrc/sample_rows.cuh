// sample_rows.cuh — a token for each row of logits by temperature, top-k,
// top-p and min-p, from given uniform numbers.
//
// Of a row, ranked by (logit descending, index ascending), with weights w =
// exp((x - max) / T): the first top_k entries stay; of those, the ones before
// which less than top_p of their mass lies; of those, the ones with w >= min_p
// (the first always stays).  What stays is a prefix of the ranking; the token
// is its first entry at which the running mass exceeds u times the prefix's.
//
// Every question is thus where a running count or mass passes a limit, and is
// answered without a sort of the row.  A cluster of blocks shares a row.  The
// weights' exponents y = (x - max) log2(e) / T fall into bins of
// 1/32 octave (what lies 64 octaves below the maximum weighs less than 2^-46 of
// any sum and is left out); a bin holds a count and the sum of 2^22 (1 - w /
// w_bin), both 32-bit integers, so masses are sums of integers: exact, and the
// same in any order.  Only the first half of the bins is filled at once; most tokens of
// a vocabulary lie below it, and are added up by threads instead of by
// additions in shared memory.  Every block sums a share of the bins for all, and where few
// entries lie up to the bin that decides, these are gathered in the first
// block, sorted and walked.  Otherwise the first block asks for more: the other
// bins and a list up to the deciding one, or each limit's bin by itself; one of more than kSrList entries is
// divided by the logits' bits, and equal logits by index.
//
// Bound: latency for few rows (loads, four barriers of the cluster, a short
// sort; 6 us more where top_k reaches below the near bins beside one token that
// holds nearly all), for many the instructions of three passes over a row from the
// caches, 53 an entry in all: 2.2 issue a cycle (integer pipe 32 % busy, DRAM 7 %),
// which wait for one another's results, additions in shared memory and barriers.
// 68 to 120 bytes a thread are spilled.  Measured on a B200 (us; graphs of calls
// on alternating inputs): a row of 128256 fp32 logits 16.9, 64 of bf16 with
// settings of their own 39.2, 256 of 32000 in fp16 without filters 28.6.
#pragma once
#include <cooperative_groups.h>
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <type_traits>

#include "common.cuh"

namespace fwb {

namespace cg = cooperative_groups;

constexpr int kSrThreads = 512, kSrBins = 2048, kSrList = 2048;
constexpr int kSrNear = 1024;              // bins filled at once
constexpr int kSrKept = 1024;              // entries of the first half of these that a block keeps a list of
constexpr uint32_t kSrSlice = 32768;       // most entries of a block: its bins' sums stay below 2^32
constexpr uint32_t kSrCluster = 8;         // most blocks of a row
constexpr float kSrUnit = 4194304.f;       // 2^22

struct SampleRowsArgs {
    const void *logits;
    uint64_t stride;
    uint32_t n_vocab, slice, vec;           // vec: rows are 16-byte aligned
    const float *u, *temp, *top_p, *min_p;  // the last three and top_k may be null
    const int32_t *top_k;
    int32_t *token;
    float *logprob;                         // may be null
};

// The entries that a round is about: bins k0..k1, of those the keys
// klo..khi, of those the indexes ilo..ihi.
struct SrRange {
    uint32_t k0, k1, klo, khi, ilo, ihi;
};
enum SrOp : uint32_t { kSrDone, kSrFar, kSrHist, kSrLow, kSrCollect };

struct SrSmem {
    uint2 bins[kSrBins];                 // {entries, the sum of what their weights lack}
    uint32_t cum_c[kSrBins];             // (first block) entries and mass up to and with a bin
    double cum_w[kSrBins];
    // (first block) the list, key << 32 | ~index, with the mass up to and with
    // an entry once sorted; before it, the sums of a bin's divisions
    union {
        unsigned long long list[kSrList];
        uint32_t sub_c[kSrBins];
    };
    union {
        double list_w[kSrList];
        double sub_w[kSrBins];
    };
    unsigned long long best[kSrCluster]; // the blocks' largest entries
    uint32_t bad[kSrCluster];
    double far[kSrCluster];              // the blocks' masses below the near bins
    unsigned long long kept[kSrKept];    // key << 32 | ~index
    uint32_t op, shift, listed, n_kept;
    SrRange range;
    uint32_t found;
    double wsum[kSrThreads / 32], steps[32];
    uint32_t csum[kSrThreads / 32];
    unsigned long long wbest[kSrThreads / 32];
    uint32_t wbad[kSrThreads / 32];
};

__device__ __forceinline__ uint32_t sr_key(float x) {
    const uint32_t u = __float_as_uint(x + 0.f);  // (-0 is 0)
    return u >> 31 ? ~u : u | 0x80000000u;
}
__device__ __forceinline__ float sr_value(uint32_t key) { return __uint_as_float(key >> 31 ? key & 0x7fffffffu : ~key); }

// A block's slice of a row: read again by every pass, from the caches after the
// first (held in registers, the passes' unrolled code spilled: 2.5 times slower).
template <typename T>
struct SrSlice {
    static constexpr uint32_t N = 16 / sizeof(T);
    const T *row;
    uint32_t begin, end, vec;
    // 16 bytes of entries from i on, those past the end -inf
    __device__ __forceinline__ uint4 load(uint32_t i) const {
        if (vec && i + N <= end) return __ldg(reinterpret_cast<const uint4 *>(row + i));
        uint32_t w[4];
#pragma unroll
        for (uint32_t j = 0; j < N; ++j) {
            if constexpr (sizeof(T) == 4) {
                w[j] = i + j < end ? __float_as_uint(row[i + j]) : 0xff800000u;
            } else {
                const uint32_t h = i + j < end ? reinterpret_cast<const uint16_t *>(row)[i + j]
                                               : std::is_same<T, __half>::value ? 0xfc00u : 0xff80u;
                w[j / 2] = j % 2 ? w[j / 2] | h << 16 : h;
            }
        }
        return make_uint4(w[0], w[1], w[2], w[3]);
    }
    // f(logit, index) for every entry, and for some of -inf past the end; U
    // loads of a thread in flight
    template <int U, typename F>
    __device__ __forceinline__ void each(F f) const {
#pragma unroll 1
        for (uint32_t i = begin + threadIdx.x * N; i < end; i += U * kSrThreads * N) {
            uint4 v[U];
#pragma unroll
            for (int m = 0; m < U; ++m) v[m] = load(i + m * kSrThreads * N);
#pragma unroll
            for (int m = 0; m < U; ++m) {
                const uint32_t w[4] = {v[m].x, v[m].y, v[m].z, v[m].w};
#pragma unroll
                for (uint32_t j = 0; j < N; ++j) {
                    float x;
                    if constexpr (sizeof(T) == 4) x = __uint_as_float(w[j]);
                    else if constexpr (std::is_same<T, __half>::value) x = __half2float(__ushort_as_half((uint16_t)(w[j / 2] >> (j % 2 * 16))));
                    else x = __uint_as_float(j % 2 ? w[j / 2] & 0xffff0000u : w[j / 2] << 16);
                    f(x, i + m * kSrThreads * N + j);
                }
            }
        }
    }
};

// A row's constants and an entry's place: its bin and what its weight lacks to
// the bin's, in units of 2^-22.  The exponent is formed as t + lo, t rounded
// and lo its error.
struct SrScale {
    float top, hi, lo;     // log2(e) / T in two parts
    float low_hi, low_lo;  // log2(min_p)
    __device__ __forceinline__ void of(float x, float &t, float &rest) const {
        const float d = x - top;
        t = d * hi;
        rest = fmaf(d, lo, fmaf(d, hi, -t));
    }
    __device__ __forceinline__ bool high(float t, float rest) const { return (t - low_hi) + (rest - low_lo) >= 0.f; }  // w >= min_p
    __device__ __forceinline__ uint32_t bin(float t) const { return (uint32_t)(t * -32.f); }
    static __device__ __forceinline__ float weight(float y) {
        float w;
        asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(w) : "f"(y));
        return w;
    }
    __device__ __forceinline__ uint32_t frac(float t, float rest, uint32_t k) const {
        return (uint32_t)fmaxf(rintf((1.f - weight(fmaf((float)k, 1.f / 32, t) + rest)) * kSrUnit), 0.f);
    }
};

// steps: 2^(-i / 32) for i below 32
__device__ __forceinline__ double sr_mass(const double *steps, uint32_t bin, uint32_t count, unsigned long long frac) {
    return steps[bin % 32] * __hiloint2double((1023 - bin / 32) << 20, 0) * ((double)count - (double)frac * (1. / 4194304));
}

// What a block does for the first one, which asked through sh.op: counts the
// entries of a range in bins, or gives them to the first block's list.
template <typename T>
__device__ __noinline__ void sr_serve(SrSmem &sh, SrSmem &first, SrSlice<T> x, SrScale s) {
    const SrRange r = sh.range;
    const uint32_t op = sh.op, shift = sh.shift;
    x.template each<2>([&](float v, uint32_t i) {
        float t, rest;
        s.of(v, t, rest);
        const uint32_t k = s.bin(t), key = sr_key(v);
        if (v == -INFINITY || k < r.k0 || k > r.k1 || key < r.klo || key > r.khi || i < r.ilo || i > r.ihi) return;
        if (op == kSrCollect) {
            const uint32_t at = atomicAdd(&first.listed, 1u);
            if (at < kSrList) first.list[at] = (unsigned long long)key << 32 | ~i;
            return;
        }
        const uint32_t at = op == kSrFar ? k : op == kSrLow ? 2 * (k - r.k0) + (s.high(t, rest) ? 0 : 1)
                            : r.klo < r.khi ? (r.khi - key) >> shift : (i - r.ilo) >> shift;
        atomicAdd(&sh.bins[at].x, 1u);
        atomicAdd(&sh.bins[at].y, s.frac(t, rest, k));
    });
}

// Inclusive sums over the block's threads, K values each.
template <int K>
__device__ __forceinline__ void sr_scan(SrSmem &sh, uint32_t (&c)[K], double (&w)[K]) {
    const uint32_t lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
#pragma unroll
    for (int i = 1; i < K; ++i) {
        c[i] += c[i - 1];
        w[i] += w[i - 1];
    }
    uint32_t cs = c[K - 1];
    double ws = w[K - 1];
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
        const uint32_t x = __shfl_up_sync(0xffffffffu, cs, d);
        const double y = __shfl_up_sync(0xffffffffu, ws, d);
        if (lane >= (uint32_t)d) {
            cs += x;
            ws += y;
        }
    }
    __syncthreads();
    if (lane == 31) {
        sh.csum[warp] = cs;
        sh.wsum[warp] = ws;
    }
    __syncthreads();
    uint32_t cb = lane < kSrThreads / 32 && lane < warp ? sh.csum[lane] : 0;
    double before = lane < kSrThreads / 32 && lane < warp ? sh.wsum[lane] : 0.;
    cb = __reduce_add_sync(0xffffffffu, cb) + cs - c[K - 1];
#pragma unroll
    for (int d = 8; d; d >>= 1) before += __shfl_xor_sync(0xffffffffu, before, d);
    before = __shfl_sync(0xffffffffu, before, 0);
    double wb = __shfl_up_sync(0xffffffffu, ws, 1);
    if (!lane) wb = 0.;
    wb += before;
#pragma unroll
    for (int i = 0; i < K; ++i) {
        c[i] += cb;
        w[i] += wb;
    }
}

template <typename T>
__global__ void __launch_bounds__(kSrThreads, 2) sample_rows_kernel(const __grid_constant__ SampleRowsArgs a) {
    extern __shared__ __align__(16) uint8_t dyn[];
    SrSmem &sh = *reinterpret_cast<SrSmem *>(dyn);
    cg::cluster_group cluster = cg::this_cluster();
    const uint32_t tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, blocks = cluster.num_blocks(),
                   rank = cluster.block_rank(), row = blockIdx.x / blocks;
    pdl_wait();
    const uint32_t begin = min(rank * a.slice, a.n_vocab);
    const SrSlice<T> x = {static_cast<const T *>(a.logits) + row * a.stride, begin, min(begin + a.slice, a.n_vocab), a.vec};
    const float temp = a.temp ? a.temp[row] : 1.f, u = a.u[row], low = a.min_p ? a.min_p[row] : 0.f;
    const double top_p = a.top_p ? (double)a.top_p[row] : 1.;
    const int32_t top_k = a.top_k ? a.top_k[row] : 0;
    for (uint32_t b = tid; b < kSrNear; b += kSrThreads) sh.bins[b] = make_uint2(0, 0);
    if (tid == 0) sh.listed = sh.n_kept = 0;

    // --- the largest entry ---
    {
        float best = -INFINITY;
        uint32_t at = 0xffffffffu, bad = 0;
        x.template each<4>([&](float v, uint32_t i) {
            bad |= !(v < INFINITY);
            if (v > best) {
                best = v;
                at = i;
            }
        });
        unsigned long long key = (unsigned long long)sr_key(best) << 32 | (at == 0xffffffffu ? 0u : ~at);
#pragma unroll
        for (int d = 16; d; d >>= 1) {
            const unsigned long long o = __shfl_xor_sync(0xffffffffu, key, d);
            key = o > key ? o : key;
        }
        bad = __any_sync(0xffffffffu, bad);
        if (lane == 0) {
            sh.wbest[warp] = key;
            sh.wbad[warp] = bad;
        }
        __syncthreads();
        if (warp == 0) {
            key = lane < kSrThreads / 32 ? sh.wbest[lane] : 0;
            bad = __any_sync(0xffffffffu, lane < kSrThreads / 32 ? sh.wbad[lane] : 0);
#pragma unroll
            for (int d = 8; d; d >>= 1) {
                const unsigned long long o = __shfl_xor_sync(0xffffffffu, key, d);
                key = o > key ? o : key;
            }
            key = __shfl_sync(0xffffffffu, key, 0);
            if (lane < blocks) {
                SrSmem &to = *cluster.map_shared_rank(&sh, lane);
                to.best[rank] = key;
                to.bad[rank] = bad;
            }
        }
    }
    SrScale s;
    cluster.barrier_arrive();
    const double scale = fmin(1.4426950408889634 / (double)temp, 1e30), low2 = low > 0.f ? log2((double)low) : 0.;
    s.hi = (float)scale;
    s.lo = (float)(scale - (double)s.hi);
    s.low_hi = (float)low2;
    s.low_lo = (float)(low2 - (double)s.low_hi);
    if (tid < 32) sh.steps[tid] = exp2((double)tid * (-1. / 32));
    cluster.barrier_wait();
    unsigned long long best = sh.best[0];
    uint32_t dead = sh.bad[0];
    for (uint32_t b = 1; b < blocks; ++b) {
        best = sh.best[b] > best ? sh.best[b] : best;
        dead |= sh.bad[b];
    }
    s.top = sr_value((uint32_t)(best >> 32));
    if (dead || s.top == -INFINITY || temp != temp || u != u || temp <= 0.f) {  // (the same in every block)
        if (rank == 0 && tid == 0) {
            const bool greedy = !dead && s.top != -INFINITY && temp <= 0.f && u == u;
            a.token[row] = greedy ? (int32_t)~(uint32_t)best : -1;
            if (a.logprob) a.logprob[row] = greedy ? 0.f : -INFINITY;
        }
        return;
    }
    // --- the near bins, and what lies below them ---
    {
        float far = 0.f;
        x.template each<2>([&](float v, uint32_t i) {
            float t, rest;
            s.of(v, t, rest);
            if (t <= kSrNear * -1.f / 32) {
                if (t > kSrBins * -1.f / 32) far += s.weight((t + 32.f) + rest);
            } else if (v != -INFINITY) {
                const uint32_t k = s.bin(t);
                atomicAdd(&sh.bins[k].x, 1u);
                atomicAdd(&sh.bins[k].y, s.frac(t, rest, k));
                if (k < kSrNear / 2) {
                    const uint32_t at = atomicAdd(&sh.n_kept, 1u);
                    if (at < kSrKept) sh.kept[at] = (unsigned long long)sr_key(v) << 32 | ~i;
                }
            }
        });
        double far_w = (double)far * (1. / 4294967296);
#pragma unroll
        for (int d = 16; d; d >>= 1) far_w += __shfl_xor_sync(0xffffffffu, far_w, d);
        if (lane == 0) sh.wsum[warp] = far_w;
        __syncthreads();
        if (tid < blocks) {
            for (int w = 1; w < kSrThreads / 32; ++w) far_w = (w == 1 ? sh.wsum[0] : far_w) + sh.wsum[w];
            cluster.map_shared_rank(&sh, tid)->far[rank] = far_w;
        }
    }
    cluster.sync();
    // Each block sums a share of the bins, for all blocks.
    {
        const uint32_t share = kSrNear / blocks;
        for (uint32_t b = tid; b < share; b += kSrThreads) {
            const uint32_t at = rank * share + b;
            uint2 v[kSrCluster];
#pragma unroll
            for (uint32_t k = 0; k < kSrCluster; ++k) v[k] = k < blocks ? cluster.map_shared_rank(&sh, k)->bins[at] : make_uint2(0, 0);
            uint32_t c = 0;
            unsigned long long f = 0;
#pragma unroll
            for (uint32_t k = 0; k < kSrCluster; ++k) {
                c += v[k].x;
                f += v[k].y;
            }
            const double w = c ? sr_mass(sh.steps, at, c, f) : 0.;
#pragma unroll
            for (uint32_t k = 0; k < kSrCluster; ++k)
                if (k < blocks) {
                    SrSmem &to = *cluster.map_shared_rank(&sh, k);
                    to.cum_c[at] = c;
                    to.cum_w[at] = w;
                }
        }
    }
    cluster.sync();

    // The bins that an operation counts in, made zeros.
    auto clear = [&](uint32_t op) {
        if (op == kSrCollect) return;
        for (uint32_t b = (op == kSrFar ? kSrNear : 0) + tid; b < kSrBins; b += kSrThreads) sh.bins[b] = make_uint2(0, 0);
        __syncthreads();
    };

    // What the first block does with the others' help.
    auto ask = [&](uint32_t op, const SrRange &r, uint32_t shift) {
        __syncthreads();
        if (tid < blocks) {
            SrSmem &to = *cluster.map_shared_rank(&sh, tid);
            to.op = op;
            to.range = r;
            to.shift = shift;
        }
        if (tid == 0) sh.listed = 0;
        cluster.sync();
        if (op == kSrDone) return;
        clear(op);
        sr_serve(sh, *cluster.map_shared_rank(&sh, 0), x, s);
        cluster.sync();
    };
    // All blocks' bins from `from` on, summed up (what lies before them is): those
    // of the row, or of the divisions of bin `of`.
    auto gather = [&](uint32_t from, uint32_t of, uint32_t *cum_c, double *cum_w) {
        uint32_t c[4];
        double w[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const uint32_t b = 4 * tid + i;
            c[i] = b == 0 && from ? cum_c[from - 1] : 0;
            w[i] = b == 0 && from ? cum_w[from - 1] : 0.;
            if (b < from) continue;
            unsigned long long f = 0;
#pragma unroll 4
            for (uint32_t k = 0; k < blocks; ++k) {
                const uint2 v = cluster.map_shared_rank(&sh, k)->bins[b];
                c[i] += v.x;
                f += v.y;
            }
            w[i] = c[i] ? sr_mass(sh.steps, of < kSrBins ? of : b, c[i], f) : 0.;
        }
        sr_scan<4>(sh, c, w);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            if (4 * tid + i < from) continue;
            cum_c[4 * tid + i] = c[i];
            cum_w[4 * tid + i] = w[i];
        }
        __syncthreads();
    };
    // The first of `bins` bins up to and with which more than `count` entries, or
    // more than `mass`, lie; without one `bins`, or with `any` the last that
    // holds any.
    auto pass = [&](const uint32_t *cum_c, const double *cum_w, uint32_t bins, bool by_count, uint32_t count, double mass, bool any) {
        if (tid == 0) sh.found = bins;
        __syncthreads();
        const uint32_t each = bins / kSrThreads;
        uint32_t at = bins;
        for (int i = each - 1; i >= 0; --i)
            if (by_count ? cum_c[each * tid + i] > count : cum_w[each * tid + i] > mass) at = each * tid + i;
        if (at < bins) atomicMin(&sh.found, at);
        __syncthreads();
        if (any && sh.found == bins) {  // (read by all before it changes again)
            __syncthreads();
            for (int i = each - 1; i >= 0; --i)
                if (cum_c[each * tid + i] == cum_c[bins - 1]) at = each * tid + i;
            if (at < bins) atomicMin(&sh.found, at);
        }
        __syncthreads();
        at = sh.found;
        __syncthreads();
        return at;
    };
    uint32_t n = 0;            // entries of the list,
    uint32_t base_c = 0;       // and what comes before it
    double base_w = 0.;
    // The list in order, with its running mass.
    auto order = [&]() {
        n = min(sh.listed, (uint32_t)kSrList);
        if (n <= 128) {  // each entry counts the larger ones
            const unsigned long long e = tid < n ? sh.list[tid] : 0;
            uint32_t larger = 0;
            if (tid < n)
                for (uint32_t i = 0; i < n; ++i) larger += sh.list[i] > e;
            __syncthreads();
            if (tid < n) sh.list[larger] = e;
            __syncthreads();
        } else {
            uint32_t size = 256;
            while (size < n) size *= 2;
            for (uint32_t i = n + tid; i < size; i += kSrThreads) sh.list[i] = 0;
            __syncthreads();
            for (uint32_t k = 2; k <= size; k *= 2)
                for (uint32_t j = k / 2; j; j /= 2) {
                    for (uint32_t p = tid; p < size / 2; p += kSrThreads) {
                        const uint32_t i = 2 * p - (p & (j - 1)), o = i + j;
                        const unsigned long long e = sh.list[i], f = sh.list[o];
                        if ((e < f) == ((i & k) == 0)) {
                            sh.list[i] = f;
                            sh.list[o] = e;
                        }
                    }
                    __syncthreads();
                }
        }
        uint32_t c[4];
        double w[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            c[i] = 0;
            w[i] = 0.;
            if (4 * tid + i < n) {
                float t, rest;
                s.of(sr_value((uint32_t)(sh.list[4 * tid + i] >> 32)), t, rest);
                const uint32_t k = s.bin(t);
                w[i] = sr_mass(sh.steps, k, 1, s.frac(t, rest, k));
            }
        }
        sr_scan<4>(sh, c, w);
#pragma unroll
        for (int i = 0; i < 4; ++i) sh.list_w[4 * tid + i] = w[i];
        __syncthreads();
    };
    // How many of the list's entries lie where f(place) holds, which holds for
    // a first part of them.
    auto prefix = [&](auto f) {
        if (tid == 0) sh.found = 0;
        __syncthreads();
        uint32_t c = 0;
        for (uint32_t i = tid; i < n; i += kSrThreads) c += f(i);
        if (c) atomicAdd(&sh.found, c);
        __syncthreads();
        c = sh.found;
        __syncthreads();
        return c;
    };
    // The list of the entries of bin k near where the running count passes
    // `count` or the running mass `mass`.
    auto near = [&](uint32_t k, bool by_count, uint32_t count, double mass) {
        SrRange r = {k, k, 0u, 0xffffffffu, 0u, 0xffffffffu};
        base_c = k ? sh.cum_c[k - 1] : 0;
        base_w = k ? sh.cum_w[k - 1] : 0.;
        uint32_t held = sh.cum_c[k] - base_c;
        while (held > kSrList) {
            // keys first, indexes where there is one key
            const bool keys = r.klo < r.khi;
            if (!keys && r.ihi >= a.n_vocab) r.ihi = a.n_vocab - 1;
            const uint32_t span = keys ? r.khi - r.klo : r.ihi - r.ilo;
            uint32_t shift = 0;
            while (span >> shift >= kSrBins) ++shift;
            ask(kSrHist, r, shift);
            gather(0, k, sh.sub_c, sh.sub_w);
            const uint32_t b = pass(sh.sub_c, sh.sub_w, kSrBins, by_count, count - base_c, mass - base_w, true);
            const uint32_t c0 = b ? sh.sub_c[b - 1] : 0;
            held = sh.sub_c[b] - c0;
            base_c += c0;
            base_w += b ? sh.sub_w[b - 1] : 0.;
            if (keys) {
                const uint32_t top = r.khi - (b << shift);
                r.klo = max(r.klo, top - min(top, (1u << shift) - 1));
                r.khi = top;
            } else {
                r.ilo += b << shift;
                r.ihi = min(r.ihi, r.ilo + (1u << shift) - 1);
            }
        }
        ask(kSrCollect, r, 0);
        order();
    };

    // --- every block: the near bins of all, and the bin in which the last filter
    // ends (without one, the draw) ---
    double total = 0.;
    {
        constexpr int K = kSrNear / kSrThreads;
        uint32_t c[K];
        double w[K];
#pragma unroll
        for (int i = 0; i < K; ++i) {
            c[i] = sh.cum_c[K * tid + i];
            w[i] = sh.cum_w[K * tid + i];
        }
        sr_scan<K>(sh, c, w);
#pragma unroll
        for (int i = 0; i < K; ++i) {
            sh.cum_c[K * tid + i] = c[i];
            sh.cum_w[K * tid + i] = w[i];
        }
        __syncthreads();
        for (uint32_t k = 0; k < blocks; ++k) total += sh.far[k];
    }
    // What lies below the near bins decides nothing where its mass is below 2^-24
    // of the row's, and is not looked through then; but for a u of 1, which asks for
    // the last entry.  A filter that may leave a part of it (top_k entries, each
    // below 2^-32 of the first) wants that part to be below 2^-20 of what there is
    // besides the first, so that a logprob near 0 keeps its digits.
    const double near_w = sh.cum_w[kSrNear - 1];
    const uint32_t near_c = sh.cum_c[kSrNear - 1];
    // the bin of weight min_p, give or take a rounding
    const uint32_t low_bin = low > 0.f ? (uint32_t)fmin(fmax(low2 * -32., 1.), kSrBins - 2.) : 0;
    const bool deep_k = top_k > 0 && (uint32_t)top_k > near_c, deep_low = low > 0.f && low_bin + 1 >= kSrNear;
    const double part = deep_k ? fmin(total, (double)((uint32_t)top_k - near_c) * (1. / 4294967296)) : total;
    const bool light = u < 1.f && (deep_k || deep_low ? part <= (near_w - 1.) * (1. / 1048576) : total <= near_w * (1. / 16777216));
    total = light && top_k > 0 ? near_w : near_w + total;
    uint32_t all = light ? near_c : 0xffffffffu, bins = kSrNear, keep_k;
    bool by_k;
    const bool by_p = top_p < 1., by_low = low > 0.f && !(light && deep_low);
    // (a u of 1 or more asks for the last entry by its rank: by their masses, whose
    // sums are rounded, entries below 2^-53 of the row's are not told apart)
    const double drawn = u >= 1.f ? INFINITY : (double)u;
    auto last_bin = [&](bool any) {
        by_k = top_k > 0 && (uint32_t)top_k < all;
        keep_k = by_k ? (uint32_t)top_k : all;
        if (by_k) return pass(sh.cum_c, sh.cum_w, bins, true, keep_k - 1, 0., any);
        uint32_t at = bins;
        if (by_p) at = pass(sh.cum_c, sh.cum_w, bins, false, 0, top_p * total, any);
        if (by_low) at = min(at, low_bin + 1);
        return by_p || by_low ? at : pass(sh.cum_c, sh.cum_w, bins, false, 0, drawn * total, any);
    };
    uint32_t far = last_bin(light);
    const bool few = far < kSrNear && sh.cum_c[far] <= kSrList;  // (the same in every block)
    if (few) {
        // they go to the first block's list
        SrSmem &first = *cluster.map_shared_rank(&sh, 0);
        auto give = [&](float v, unsigned long long entry) {
            float t, rest;
            s.of(v, t, rest);
            if (s.bin(t) <= far && v != -INFINITY) first.list[atomicAdd(&first.listed, 1u)] = entry;
        };
        const uint32_t n = sh.n_kept;
        if (far < kSrNear / 2 && n <= kSrKept)
            for (uint32_t i = tid; i < n; i += kSrThreads) give(sr_value((uint32_t)(sh.kept[i] >> 32)), sh.kept[i]);
        else
            x.template each<2>([&](float v, uint32_t i) { give(v, (unsigned long long)sr_key(v) << 32 | ~i); });
    }
    cluster.sync();
    if (rank != 0) {
        while (!few) {
            cluster.sync();  // the first block has asked
            if (sh.op == kSrDone) break;
            clear(sh.op);
            sr_serve(sh, *cluster.map_shared_rank(&sh, 0), x, s);
            cluster.sync();
        }
        return;
    }

    // --- the first block ---
    uint32_t pick = 0;     // the token's place in the list
    double kept = total;   // mass of what the filters leave
    // All the filters and the draw on the list of what stands up to the last's bin.
    auto walk = [&]() {
        order();
        uint32_t stay = by_k ? keep_k : n;
        if (by_k) kept = sh.list_w[keep_k - 1];
        if (by_p) {
            const double limit = top_p * kept;
            stay = min(stay, prefix([&](uint32_t i) { return i == 0 || sh.list_w[i - 1] < limit; }));
        }
        if (by_low)
            stay = min(stay, prefix([&](uint32_t i) {
                           float t, rest;
                           s.of(sr_value((uint32_t)(sh.list[i] >> 32)), t, rest);
                           return i == 0 || s.high(t, rest);
                       }));
        if (by_k || by_p || by_low) kept = sh.list_w[stay - 1];
        const double limit = drawn * kept;
        pick = min(prefix([&](uint32_t i) { return sh.list_w[i] <= limit; }), stay - 1);
    };
    bool listed = few;
    if (few) {
        walk();
    } else {
        if (far == kSrNear) {  // below the near bins: all of them
            ask(kSrFar, {kSrNear, kSrBins - 1, 0u, 0xffffffffu, 0u, 0xffffffffu}, 0);
            gather(kSrNear, kSrBins, sh.cum_c, sh.cum_w);
            bins = kSrBins;
            all = sh.cum_c[kSrBins - 1];
            kept = total = sh.cum_w[kSrBins - 1];
            far = last_bin(true);
            if (sh.cum_c[far] <= kSrList) {
                ask(kSrCollect, {0, far, 0u, 0xffffffffu, 0u, 0xffffffffu}, 0);
                walk();
                listed = true;
            }
        }
    }
    if (!listed) {
        // each filter's end by itself, and the draw
        uint32_t stay = keep_k;
        if (by_k) {
            near(far, true, keep_k - 1, 0.);
            kept = base_w + sh.list_w[keep_k - 1 - base_c];
        }
        if (by_p) {
            const double limit = top_p * kept;
            near(pass(sh.cum_c, sh.cum_w, bins, false, 0, limit, true), false, 0, limit);
            const uint32_t c = prefix([&](uint32_t i) { return base_c + i == 0 || base_w + (i ? sh.list_w[i - 1] : 0.) < limit; });
            if (base_c + c < stay) {
                stay = base_c + c;
                kept = base_w + (c ? sh.list_w[c - 1] : 0.);
            }
        }
        if (by_low && low_bin <= far + 1) {  // (else it leaves all that the others left)
            const uint32_t k0 = low_bin - 1;
            ask(kSrLow, {k0, k0 + 2, 0u, 0xffffffffu, 0u, 0xffffffffu}, 0);
            if (tid < 3) {
                unsigned long long f = 0;
                uint32_t c = 0;
                for (uint32_t k = 0; k < blocks; ++k) {
                    const uint2 v = cluster.map_shared_rank(&sh, k)->bins[2 * tid];
                    c += v.x;
                    f += v.y;
                }
                sh.csum[tid] = c;
                sh.wsum[tid] = sr_mass(sh.steps, k0 + tid, c, f);
            }
            __syncthreads();
            const uint32_t c = (k0 ? sh.cum_c[k0 - 1] : 0) + sh.csum[0] + sh.csum[1] + sh.csum[2];
            const double w = (k0 ? sh.cum_w[k0 - 1] : 0.) + sh.wsum[0] + sh.wsum[1] + sh.wsum[2];
            if (c < stay) {
                stay = max(c, 1u);
                kept = c ? w : 1.;  // (the first entry's weight is 1)
            }
            __syncthreads();
        }
        bool last = u >= 1.f;
        if (!last) {
            const double limit = drawn * kept;
            near(pass(sh.cum_c, sh.cum_w, bins, false, 0, limit, true), false, 0, limit);
            // (the bin's sum and the list's are rounded apart: the limit may lie between them, past the list)
            pick = min(prefix([&](uint32_t i) { return base_w + sh.list_w[i] <= limit; }), n - 1);
            last = base_c + pick >= stay;
        }
        if (last) {
            near(pass(sh.cum_c, sh.cum_w, bins, true, stay - 1, 0., true), true, stay - 1, 0.);
            pick = stay - 1 - base_c;
        }
    }
    if (tid == 0) {
        const unsigned long long e = sh.list[pick];
        a.token[row] = (int32_t)~(uint32_t)e;
        if (a.logprob) {  // its own weight: in the running mass it may be below the last bit
            float t, rest;
            s.of(sr_value((uint32_t)(e >> 32)), t, rest);
            const uint32_t k = s.bin(t);
            a.logprob[row] = (float)log(sr_mass(sh.steps, k, 1, s.frac(t, rest, k)) / kept);
        }
    }
    if (!few) ask(kSrDone, {}, 0);
}

}  // namespace fwb
