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
// answered without a sort.  A cluster of blocks shares a row.  The weights'
// exponents y = (x - max) log2(e) / T fall into 2048 bins of 1/32 octave (what
// lies 64 octaves below the maximum weighs less than 2^-46 of any sum and is
// left out); a bin holds a count and the sum of 2^22 (1 - w / w_bin), both
// 32-bit integers, so masses are sums of integers: exact, and the same in any
// order.  The first block scans the bins, and only the entries of the bin
// where a limit falls (or, where few entries come before it, of all bins up to
// there) are gathered, sorted and walked.  A bin of more than kSrList entries
// is first divided again by the logits' bits, and equal logits by index.
//
// Bound: latency for few rows (a row is three or four rounds of the cluster),
// the shared-memory additions for many.
#pragma once
#include <cooperative_groups.h>
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "common.cuh"

namespace fwb {

namespace cg = cooperative_groups;

constexpr int kSrThreads = 512, kSrBins = 2048, kSrList = 2048;
constexpr uint32_t kSrSlice = 32768;       // most entries of a block: its bins' sums stay below 2^32
constexpr uint32_t kSrCluster = 8;         // most blocks of a row
constexpr float kSrUnit = 4194304.f;       // 2^22

struct SampleRowsArgs {
    const void *logits;
    uint64_t stride;
    uint32_t n_vocab, slice;
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
enum SrOp : uint32_t { kSrDone, kSrHist, kSrLow, kSrCollect };

struct SrSmem {
    uint32_t count[kSrBins], frac[kSrBins];
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
    uint32_t op, shift, listed;
    SrRange range;
    uint32_t found;
    double wsum[kSrThreads / 32];
    uint32_t csum[kSrThreads / 32];
    unsigned long long wbest[kSrThreads / 32];
    uint32_t wbad[kSrThreads / 32];
};

__device__ __forceinline__ uint32_t sr_key(float x) {
    const uint32_t u = __float_as_uint(x + 0.f);  // (-0 is 0)
    return u >> 31 ? ~u : u | 0x80000000u;
}
__device__ __forceinline__ float sr_value(uint32_t key) { return __uint_as_float(key >> 31 ? key & 0x7fffffffu : ~key); }

template <typename T> __device__ __forceinline__ float sr_float(T x);
template <> __device__ __forceinline__ float sr_float<float>(float x) { return x; }
template <> __device__ __forceinline__ float sr_float<__half>(__half x) { return __half2float(x); }
template <> __device__ __forceinline__ float sr_float<__nv_bfloat16>(__nv_bfloat16 x) { return __bfloat162float(x); }

// f(logit, index) for every entry of this block's slice.  VEC: 16-byte loads.
template <typename T, bool VEC, typename F>
__device__ __forceinline__ void sr_each(const T *row, uint32_t begin, uint32_t end, F f) {
    if constexpr (VEC) {
        constexpr uint32_t N = 16 / sizeof(T);
        const uint32_t whole = begin + (end - begin) / N * N;  // (begin is a multiple of N)
#pragma unroll 2
        for (uint32_t i = begin + threadIdx.x * N; i < whole; i += kSrThreads * N) {
            const uint4 v = *reinterpret_cast<const uint4 *>(row + i);
            const T *x = reinterpret_cast<const T *>(&v);
#pragma unroll
            for (uint32_t j = 0; j < N; ++j) f(sr_float<T>(x[j]), i + j);
        }
        for (uint32_t i = whole + threadIdx.x; i < end; i += kSrThreads) f(sr_float<T>(row[i]), i);
    } else {
        for (uint32_t i = begin + threadIdx.x; i < end; i += kSrThreads) f(sr_float<T>(row[i]), i);
    }
}

// A row's constants and an entry's place: its bin and what its weight lacks to
// the bin's, in units of 2^-22.  The exponent is formed as t + lo, t rounded
// and lo its error.
struct SrScale {
    float top, hi, lo;  // log2(e) / T in two parts
    __device__ __forceinline__ void of(float x, float &t, float &rest) const {
        const float d = x - top;
        t = d * hi;
        rest = fmaf(d, lo, fmaf(d, hi, -t));
    }
    __device__ __forceinline__ uint32_t bin(float t) const { return (uint32_t)(t * -32.f); }
    __device__ __forceinline__ uint32_t frac(float t, float rest, uint32_t k) const {
        float w;
        asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(w) : "f"(fmaf((float)k, 1.f / 32, t) + rest));
        return (uint32_t)fmaxf(rintf((1.f - w) * kSrUnit), 0.f);
    }
};

__device__ __forceinline__ double sr_mass(uint32_t bin, uint32_t count, unsigned long long frac) {
    return exp2((double)bin * (-1. / 32)) * ((double)count - (double)frac * (1. / 4194304));
}

// Inclusive sums over the block's threads, four values each.
__device__ __forceinline__ void sr_scan(SrSmem &sh, uint32_t (&c)[4], double (&w)[4]) {
    const uint32_t lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
#pragma unroll
    for (int i = 1; i < 4; ++i) {
        c[i] += c[i - 1];
        w[i] += w[i - 1];
    }
    uint32_t cs = c[3];
    double ws = w[3];
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
    uint32_t cb = cs - c[3];
    double wb = __shfl_up_sync(0xffffffffu, ws, 1);
    if (!lane) wb = 0.;
    double before = 0.;
    for (uint32_t v = 0; v < warp; ++v) {
        cb += sh.csum[v];
        before += sh.wsum[v];
    }
    wb += before;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        c[i] += cb;
        w[i] += wb;
    }
}

template <typename T, bool VEC>
__global__ void __launch_bounds__(kSrThreads) sample_rows_kernel(const __grid_constant__ SampleRowsArgs a) {
    extern __shared__ __align__(16) uint8_t dyn[];
    SrSmem &sh = *reinterpret_cast<SrSmem *>(dyn);
    cg::cluster_group cluster = cg::this_cluster();
    const uint32_t tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, blocks = cluster.num_blocks(),
                   rank = cluster.block_rank(), row = blockIdx.x / blocks;
    pdl_wait();
    const T *const x = static_cast<const T *>(a.logits) + row * a.stride;
    const uint32_t begin = min(rank * a.slice, a.n_vocab), end = min(begin + a.slice, a.n_vocab);

    // --- the largest entry ---
    {
        float best = -INFINITY;
        uint32_t at = 0xffffffffu, bad = 0;
        sr_each<T, VEC>(x, begin, end, [&](float v, uint32_t i) {
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
        for (uint32_t b = tid; b < kSrBins; b += kSrThreads) sh.count[b] = sh.frac[b] = 0;
        if (tid == 0) sh.listed = 0;
        __syncthreads();
        if (tid < blocks) {
            key = sh.wbest[0];
            bad = sh.wbad[0];
            for (int w = 1; w < kSrThreads / 32; ++w) {
                key = sh.wbest[w] > key ? sh.wbest[w] : key;
                bad |= sh.wbad[w];
            }
            SrSmem &to = *cluster.map_shared_rank(&sh, tid);
            to.best[rank] = key;
            to.bad[rank] = bad;
        }
        cluster.sync();
    }
    unsigned long long best = sh.best[0];
    uint32_t dead = sh.bad[0];
    for (uint32_t b = 1; b < blocks; ++b) {
        best = sh.best[b] > best ? sh.best[b] : best;
        dead |= sh.bad[b];
    }
    SrScale s;
    s.top = sr_value((uint32_t)(best >> 32));
    const float temp = a.temp ? a.temp[row] : 1.f, u = a.u[row];
    if (dead || s.top == -INFINITY || temp != temp || u != u || temp <= 0.f) {  // (the same in every block)
        if (rank == 0 && tid == 0) {
            const bool greedy = !dead && s.top != -INFINITY && temp <= 0.f;
            a.token[row] = greedy ? (int32_t)~(uint32_t)best : -1;
            if (a.logprob) a.logprob[row] = greedy ? 0.f : -INFINITY;
        }
        return;
    }
    {
        const double c = fmin(1.4426950408889634 / (double)temp, 1e30);
        s.hi = (float)c;
        s.lo = (float)(c - (double)s.hi);
    }

    // --- the row's bins ---
    sr_each<T, VEC>(x, begin, end, [&](float v, uint32_t) {
        float t, rest;
        s.of(v, t, rest);
        const uint32_t k = s.bin(t);
        if (k < kSrBins && v != -INFINITY) {
            atomicAdd(&sh.count[k], 1u);
            atomicAdd(&sh.frac[k], s.frac(t, rest, k));
        }
    });
    cluster.sync();

    // What the blocks do for the first one, which asks through sh.op.
    const float low = a.min_p ? a.min_p[row] : 0.f;
    const double low2 = low > 0.f ? log2((double)low) : 0.;
    const float low_hi = (float)low2, low_lo = (float)(low2 - (double)low_hi);
    auto high = [&](float t, float rest) { return (t - low_hi) + (rest - low_lo) >= 0.f; };  // w >= min_p
    auto serve = [&]() {
        const SrRange r = sh.range;
        const uint32_t op = sh.op, shift = sh.shift;
        SrSmem &first = *cluster.map_shared_rank(&sh, 0);
        sr_each<T, VEC>(x, begin, end, [&](float v, uint32_t i) {
            float t, rest;
            s.of(v, t, rest);
            const uint32_t k = s.bin(t);
            if (k < r.k0 || k > r.k1 || v == -INFINITY) return;
            if (op == kSrLow) {
                const uint32_t at = 2 * (k - r.k0) + (high(t, rest) ? 0 : 1);
                atomicAdd(&sh.count[at], 1u);
                atomicAdd(&sh.frac[at], s.frac(t, rest, k));
                return;
            }
            const uint32_t key = sr_key(v);
            if (key < r.klo || key > r.khi || i < r.ilo || i > r.ihi) return;
            if (op == kSrCollect) {
                const uint32_t at = atomicAdd(&first.listed, 1u);
                if (at < kSrList) first.list[at] = (unsigned long long)key << 32 | ~i;
            } else {
                const uint32_t at = r.klo < r.khi ? (r.khi - key) >> shift : (i - r.ilo) >> shift;
                atomicAdd(&sh.count[at], 1u);
                atomicAdd(&sh.frac[at], s.frac(t, rest, k));
            }
        });
    };
    if (rank != 0) {
        while (true) {
            cluster.sync();  // the first block has asked
            if (sh.op == kSrDone) break;
            if (sh.op != kSrCollect) {
                for (uint32_t b = tid; b < kSrBins; b += kSrThreads) sh.count[b] = sh.frac[b] = 0;
                __syncthreads();
            }
            serve();
            cluster.sync();
        }
        return;
    }

    // --- the first block ---
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
        if (op != kSrCollect) {
            for (uint32_t b = tid; b < kSrBins; b += kSrThreads) sh.count[b] = sh.frac[b] = 0;
            __syncthreads();
        }
        serve();
        cluster.sync();
    };
    // All blocks' bins, summed up: those of the row, or of the divisions of bin `of`.
    auto gather = [&](uint32_t of, uint32_t *cum_c, double *cum_w) {
        uint32_t c[4];
        double w[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const uint32_t b = 4 * tid + i;
            unsigned long long f = 0;
            c[i] = 0;
            for (uint32_t k = 0; k < blocks; ++k) {
                const SrSmem &from = *cluster.map_shared_rank(&sh, k);
                c[i] += from.count[b];
                f += from.frac[b];
            }
            w[i] = c[i] ? sr_mass(of < kSrBins ? of : b, c[i], f) : 0.;
        }
        sr_scan(sh, c, w);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            cum_c[4 * tid + i] = c[i];
            cum_w[4 * tid + i] = w[i];
        }
        __syncthreads();
    };
    // The first bin up to and with which more than `count` entries, or more
    // than `mass`, lie (without one, the last that holds any).
    auto pass = [&](const uint32_t *cum_c, const double *cum_w, bool by_count, uint32_t count, double mass) {
        if (tid == 0) sh.found = kSrBins;
        __syncthreads();
        uint32_t at = kSrBins;
        for (int i = 3; i >= 0; --i)
            if (by_count ? cum_c[4 * tid + i] > count : cum_w[4 * tid + i] > mass) at = 4 * tid + i;
        if (at < kSrBins) atomicMin(&sh.found, at);
        __syncthreads();
        if (sh.found == kSrBins) {  // (read by all before it changes again)
            __syncthreads();
            for (int i = 3; i >= 0; --i)
                if (cum_c[4 * tid + i] == cum_c[kSrBins - 1]) at = 4 * tid + i;
            if (at < kSrBins) atomicMin(&sh.found, at);
        }
        __syncthreads();
        at = sh.found;
        __syncthreads();
        return at;
    };
    uint32_t n = 0;            // entries of the list,
    uint32_t base_c = 0;       // and what comes before it
    double base_w = 0.;
    // The entries of a range in order, with their running mass.
    auto collect = [&](const SrRange &r) {
        ask(kSrCollect, r, 0);
        n = min(sh.listed, (uint32_t)kSrList);
        uint32_t size = 32;
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
                w[i] = sr_mass(k, 1, s.frac(t, rest, k));
            }
        }
        sr_scan(sh, c, w);
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
            gather(k, sh.sub_c, sh.sub_w);
            const uint32_t b = pass(sh.sub_c, sh.sub_w, by_count, count - base_c, mass - base_w);
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
        collect(r);
    };

    gather(kSrBins, sh.cum_c, sh.cum_w);
    const uint32_t all = sh.cum_c[kSrBins - 1];
    const double total = sh.cum_w[kSrBins - 1];
    const int32_t top_k = a.top_k ? a.top_k[row] : 0;
    const double top_p = a.top_p ? (double)a.top_p[row] : 1.;
    const bool by_k = top_k > 0 && (uint32_t)top_k < all, by_p = top_p < 1., by_low = low > 0.f;
    const uint32_t keep_k = by_k ? (uint32_t)top_k : all;
    // the bin of weight min_p, give or take a rounding
    const uint32_t low_bin = by_low ? (uint32_t)fmin(fmax(low2 * -32., 1.), kSrBins - 2.) : 0;
    // the bin in which the last filter ends (without one, the draw)
    uint32_t far;
    if (by_k) {
        far = pass(sh.cum_c, sh.cum_w, true, keep_k - 1, 0.);
    } else if (by_p) {
        far = pass(sh.cum_c, sh.cum_w, false, 0, top_p * total);
        if (by_low) far = min(far, low_bin + 1);
    } else if (by_low) {
        far = low_bin + 1;
    } else {
        far = pass(sh.cum_c, sh.cum_w, false, 0, (double)u * total);
    }
    uint32_t pick = 0;     // the token's place in the list
    double kept = total;   // mass of what the filters leave
    if (sh.cum_c[far] <= kSrList) {
        // few entries: all of them up to there in one list
        collect({0u, far, 0u, 0xffffffffu, 0u, 0xffffffffu});
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
                           return i == 0 || high(t, rest);
                       }));
        if (by_k || by_p || by_low) kept = sh.list_w[stay - 1];
        const double limit = (double)u * kept;
        pick = min(prefix([&](uint32_t i) { return sh.list_w[i] <= limit; }), stay - 1);
    } else {
        // each filter's end by itself, then the draw
        uint32_t stay = keep_k;
        if (by_k) {
            near(far, true, keep_k - 1, 0.);
            kept = base_w + sh.list_w[keep_k - 1 - base_c];
        }
        if (by_p) {
            const double limit = top_p * kept;
            near(pass(sh.cum_c, sh.cum_w, false, 0, limit), false, 0, limit);
            const uint32_t c = prefix([&](uint32_t i) { return base_c + i == 0 || base_w + (i ? sh.list_w[i - 1] : 0.) < limit; });
            if (base_c + c < stay) {
                stay = base_c + c;
                kept = base_w + (c ? sh.list_w[c - 1] : 0.);
            }
        }
        if (by_low) {
            const uint32_t k0 = low_bin - 1;
            ask(kSrLow, {k0, k0 + 2, 0u, 0xffffffffu, 0u, 0xffffffffu}, 0);
            if (tid < 3) {
                unsigned long long f = 0;
                uint32_t c = 0;
                for (uint32_t k = 0; k < blocks; ++k) {
                    const SrSmem &from = *cluster.map_shared_rank(&sh, k);
                    c += from.count[2 * tid];
                    f += from.frac[2 * tid];
                }
                sh.csum[tid] = c;
                sh.wsum[tid] = sr_mass(k0 + tid, c, f);
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
        const double limit = (double)u * kept;
        near(pass(sh.cum_c, sh.cum_w, false, 0, limit), false, 0, limit);
        pick = prefix([&](uint32_t i) { return base_w + sh.list_w[i] <= limit; });
        if (base_c + pick >= stay) {  // u is 1, or rounding: the last that stays
            near(pass(sh.cum_c, sh.cum_w, true, stay - 1, 0.), true, stay - 1, 0.);
            pick = stay - 1 - base_c;
        }
    }
    const uint32_t index = ~(uint32_t)sh.list[pick];
    if (tid == 0) {
        const double w = sh.list_w[pick] - (pick ? sh.list_w[pick - 1] : 0.);
        a.token[row] = (int32_t)index;
        if (a.logprob) a.logprob[row] = (float)log(w / kept);
    }
    ask(kSrDone, {}, 0);
}

}  // namespace fwb
