// kv4_append.cuh — new tokens into the paged cache of 4-bit keys and values,
// and positions of it back as values.
//
// Queries and keys are rotated by position (rope.c:28-53; pairs of neighbours
// as there, or of the two halves of a head):
//
//     (a, b) -> (a cos - b sin, a sin + b cos)
//
// Keys then, and values as they are, become blocks of 32 in 4 bits: with m the
// value of the largest magnitude (the positive one of two), d = fp16(-m / 8)
// and the code floor(y / d + 8.5), held to 0..15: m itself stands at -8 d.
// These are Q4_0's values; the scale that is stored, not the one before its
// rounding, decides the codes.  A key's y is the fp32 value nearest to the
// exact rotation (the products are exact in 64 bits), and codes are decided by
// exact comparisons, so that a cache's content does not depend on how a sum was
// rounded.
//
// Bound: the launch for steps, the latency of loads for prompts.  Four lanes hold a block, eight
// values each: its scale is two shuffles of each extreme, a lane has a whole
// word of a key's codes, and every store goes to bytes of this position alone.
// Measured on a B200 (us; graphs of calls on alternating inputs), to append and to
// read back: 64 fp16 sequences of one token, 32 heads of 128 on 8, 3.0 and 2.1; a
// prompt of 2048 fp32 tokens 20.9 and 8.9; 7 bf16 chunks of 333
// tokens, 64 heads on 8, 23.5 and 9.9: 3.5 and 3.0 TB/s together, the ends of two
// launches in them.  Of the prompt's append half of the stall cycles wait for loads,
// at 64 registers and 42 % of the warps (2.0 instructions a cycle, integer pipe 37 %,
// the products in 64 bits 1 %); the read spends its time on the indexes of four
// values a thread (four divisions each) and the same waits (2.6 a cycle).
#pragma once
#include "kv4_format.cuh"

namespace fwb {

constexpr int kKpThreads = 128;

struct Kv4Rows {  // [n_seq][n_query][heads][head_dim], strides in elements
    const void *p;
    uint64_t seq, tok, head;
};

struct Kv4AppendArgs {
    Kv4Rows q, k, v, q_out;  // (q_out.p is written)
    uint8_t *cache;
    const int32_t *pages, *len, *n_new;
    const float *cos, *sin;  // [n_pos][hd / 2], or null: not rotated
    uint64_t pages_seq;
    uint32_t n_seq, n_query, n_head, n_kv, hd, page_log2, n_page, max_pages, n_pos;
    uint32_t by_part, by_blocks;  // 2^32 over the chunk pairs of a query row, and the blocks of a row, rounded up (0: over 1)
    uint32_t *err;
};

// Position of token t of a sequence; -1 if it has none or it does not fit.
__device__ __forceinline__ int32_t kp_position(const Kv4AppendArgs &a, uint32_t seq, uint32_t t, uint32_t &bad) {
    const int32_t fresh = a.n_new ? min(max(a.n_new[seq], 0), (int32_t)a.n_query) : (int32_t)a.n_query;
    if ((int32_t)t >= fresh) return -1;
    const int64_t pos = (int64_t)a.len[seq] - fresh + t;
    if (pos < 0) return -1;
    if (pos >= (int64_t)a.max_pages << a.page_log2 || (a.cos && pos >= a.n_pos)) {
        bad |= kKvBadPosition;
        return -1;
    }
    return (int32_t)pos;
}

enum KpTurn { kKpNone, kKpNeighbours, kKpHalves };

// x cos - y sin, to fp32: with two roundings for queries, with one for keys.
template <bool EXACT>
__device__ __forceinline__ float kp_turn(float x, float c, float y, float s) {
    if constexpr (EXACT) return (float)((double)x * c - (double)y * s);
    else return fmaf(x, c, -(y * s));
}

// Two chunks of 16 bytes of a query row, half a row apart: whole pairs either
// way, so that a row may be turned in place.
template <typename T>
struct KpQuery {
    static constexpr int N = 16 / sizeof(T);
    float x[N], y[N];
    uint32_t h, j;
};
template <typename T>
__device__ __forceinline__ void kp_chunk(const void *p, uint64_t at, float (&x)[16 / sizeof(T)]) {
    if constexpr (sizeof(T) == 2) {
        kv4_load8<T>(p, at, x);
    } else {
        const float4 v = kv4_load4<T>(p, at);
        x[0] = v.x; x[1] = v.y; x[2] = v.z; x[3] = v.w;
    }
}
template <typename T>
__device__ __forceinline__ void kp_query_load(const Kv4AppendArgs &a, uint32_t i, uint64_t from, KpQuery<T> &q) {
    const uint32_t part = a.hd / (2 * q.N);
    q.h = part == 1 ? i : __umulhi(i, a.by_part);
    q.j = i - q.h * part;
    if (q.h < a.n_head) {
        kp_chunk<T>(a.q.p, from + q.h * a.q.head + q.N * q.j, q.x);
        kp_chunk<T>(a.q.p, from + q.h * a.q.head + q.N * q.j + a.hd / 2, q.y);
    }
}
template <typename T>
__device__ __forceinline__ void kp_chunk_store(void *p, uint64_t at, const float (&x)[16 / sizeof(T)]) {
    if constexpr (sizeof(T) == 2) kv4_store8<T>(p, at, x);
    else kv4_store4<T>(p, at, make_float4(x[0], x[1], x[2], x[3]));
}
// M angles' cosines and sines.
template <int M>
__device__ __forceinline__ void kp_angles(const Kv4AppendArgs &a, uint64_t at, float (&c)[M], float (&s)[M]) {
    if constexpr (M == 2) {
        const float2 u = *reinterpret_cast<const float2 *>(a.cos + at), v = *reinterpret_cast<const float2 *>(a.sin + at);
        c[0] = u.x; c[1] = u.y; s[0] = v.x; s[1] = v.y;
    } else {
#pragma unroll
        for (int m = 0; m < M; m += 4) {
            const float4 u = kv4_load4<float>(a.cos, at + m), v = kv4_load4<float>(a.sin, at + m);
            c[m] = u.x; c[m + 1] = u.y; c[m + 2] = u.z; c[m + 3] = u.w;
            s[m] = v.x; s[m + 1] = v.y; s[m + 2] = v.z; s[m + 3] = v.w;
        }
    }
}
// Neighbours turned, in a chunk of N values from dimension d on.
template <bool EXACT, int N>
__device__ __forceinline__ void kp_neighbours(const Kv4AppendArgs &a, uint32_t pos, uint32_t d, float (&x)[N]) {
    float c[N / 2], s[N / 2];
    kp_angles(a, (uint64_t)pos * (a.hd / 2) + d / 2, c, s);
#pragma unroll
    for (int m = 0; m < N / 2; ++m) {
        const float u = kp_turn<EXACT>(x[2 * m], c[m], x[2 * m + 1], s[m]);
        x[2 * m + 1] = kp_turn<EXACT>(x[2 * m + 1], c[m], x[2 * m], -s[m]);
        x[2 * m] = u;
    }
}
template <typename T, KpTurn TURN>
__device__ __forceinline__ void kp_query_store(const Kv4AppendArgs &a, KpQuery<T> &q, uint64_t to, uint32_t pos) {
    if (q.h >= a.n_head) return;
    constexpr int N = KpQuery<T>::N;
    if constexpr (TURN == kKpNeighbours) {
        kp_neighbours<false>(a, pos, N * q.j, q.x);
        kp_neighbours<false>(a, pos, N * q.j + a.hd / 2, q.y);
    } else if constexpr (TURN == kKpHalves) {
        float c[N], s[N];
        kp_angles(a, (uint64_t)pos * (a.hd / 2) + N * q.j, c, s);
#pragma unroll
        for (int m = 0; m < N; ++m) {
            const float u = kp_turn<false>(q.x[m], c[m], q.y[m], s[m]);
            q.y[m] = kp_turn<false>(q.y[m], c[m], q.x[m], -s[m]);
            q.x[m] = u;
        }
    }
    kp_chunk_store<T>(const_cast<void *>(a.q_out.p), to + q.h * a.q_out.head + N * q.j, q.x);
    kp_chunk_store<T>(const_cast<void *>(a.q_out.p), to + q.h * a.q_out.head + N * q.j + a.hd / 2, q.y);
}

// The code of y: floor(y / d + 8.5) held to 0..15.  The integer nearest to y *
// (1 / d) is one off at most; what is left of y beyond its code is exact in
// fp32 (codes have 4 bits, d has 11), and a comparison with d / 2 decides.
// a = |d| and inv = 1 / a, or where d is 0 the largest float and 0.
__device__ __forceinline__ uint32_t kp_code(float y, float d, float a, float inv) {
    const float z = d < 0.f ? -y : y, t = fminf(fmaxf(z * inv, -9.f), 9.f), n = rintf(t), left = fmaf(-n, a, z), half = 0.5f * a;
    const int k = (int)n + 8 + (left >= half ? 1 : 0) - (left < -half ? 1 : 0);
    return (uint32_t)min(max(k, 0), 15);
}

// Eight values of a block of a key or value row (zeros past its end), and where
// halves are turned the eight that they pair with.
struct KpBlock {
    float x[8], z[8];
    uint32_t head, b;
    bool value;
};
template <typename T, KpTurn TURN>
__device__ __forceinline__ void kp_block_load(const Kv4AppendArgs &a, uint32_t i, uint32_t seq, uint32_t t, bool is, KpBlock &k) {
    const uint32_t nb = kv4_blocks(a.hd), unit = i / 4, h = nb == 1 ? unit : __umulhi(unit, a.by_blocks);
    k.value = h >= a.n_kv;
    k.head = k.value ? h - a.n_kv : h;
    k.b = unit - h * nb;
    const uint32_t d0 = 32 * k.b + 8 * (i % 4);
#pragma unroll
    for (int m = 0; m < 8; ++m) k.x[m] = 0.f;
    if (is && d0 < a.hd) {
        const Kv4Rows &src = k.value ? a.v : a.k;
        const uint64_t from = seq * src.seq + t * src.tok + k.head * src.head;
        kv4_load8<T>(src.p, from + d0, k.x);
        if constexpr (TURN == kKpHalves)
            if (!k.value) kv4_load8<T>(src.p, from + (d0 >= a.hd / 2 ? d0 - a.hd / 2 : d0 + a.hd / 2), k.z);
    }
}
// The block rotated, quantised and stored, by the four lanes that hold it (all
// of a warp's lanes come here together; is: whether this one holds any).
template <KpTurn TURN>
__device__ __forceinline__ void kp_block_store(const Kv4AppendArgs &a, KpBlock &k, uint32_t i, uint32_t page, uint32_t pos, bool is) {
    const uint32_t nb = kv4_blocks(a.hd), j = i % 4, d0 = 32 * k.b + 8 * j;
    float (&y)[8] = k.x;
    if (TURN != kKpNone && is && !k.value && d0 < a.hd) {
        if constexpr (TURN == kKpHalves) {
            const uint64_t at = (uint64_t)pos * (a.hd / 2);
            const bool upper = d0 >= a.hd / 2;
            float c[8], s[8];
            kp_angles(a, at + (upper ? d0 - a.hd / 2 : d0), c, s);
#pragma unroll
            for (int m = 0; m < 8; ++m) y[m] = kp_turn<true>(y[m], c[m], k.z[m], upper ? -s[m] : s[m]);
        } else {
            kp_neighbours<true>(a, pos, d0, y);
        }
    }
    float hi = y[0], lo = y[0], odd = y[0] * 0.f;  // odd: NaN where something is not finite
#pragma unroll
    for (int m = 1; m < 8; ++m) {
        hi = fmaxf(hi, y[m]);
        lo = fminf(lo, y[m]);
        odd = fmaf(y[m], 0.f, odd);
    }
#pragma unroll
    for (int m = 1; m < 4; m <<= 1) {
        hi = fmaxf(hi, __shfl_xor_sync(0xffffffffu, hi, m));
        lo = fminf(lo, __shfl_xor_sync(0xffffffffu, lo, m));
        odd += __shfl_xor_sync(0xffffffffu, odd, m);
    }
    // a block with a value that is not finite is NaN throughout; past what fp16
    // scales reach (|m| > 524032) values are held to the largest
    const bool bad = odd != odd;
    const __half dh = bad ? __ushort_as_half(0x7fff)
                          : __float2half_rn(fminf(fmaxf((hi >= -lo ? hi : lo) * -0.125f, -65504.f), 65504.f));
    const float d = bad ? 0.f : __half2float(dh), mag = d == 0.f ? 3e38f : fabsf(d), inv = d == 0.f ? 0.f : __frcp_rn(mag);
    uint32_t word = 0, code[8];
#pragma unroll
    for (int m = 0; m < 8; ++m) {
        code[m] = bad ? 8u : kp_code(y[m], d, mag, inv);
        word |= code[m] << (4 * (m / 2) + 16 * (m % 2));
    }
    if (!is) return;
    const uint32_t in = pos & ((1u << a.page_log2) - 1), p = in % kKvTile;
    uint8_t *tile = a.cache + ((((uint64_t)page * a.n_kv + k.head) << (a.page_log2 - 4)) + in / kKvTile) * kv4_tile(nb) +
                    (k.value ? kv4_codes(nb) + kv4_scales(nb) : 0);
    if (k.value) {
        uint8_t *to = tile + p * 16 * nb + 2 * k.b + (2 * j ^ (p & 2 ? 4u : 0u)) * 2 * nb;  // and the unit after it
        *reinterpret_cast<uint16_t *>(to) = (uint16_t)(code[0] | code[1] << 4 | code[2] << 8 | code[3] << 12);
        *reinterpret_cast<uint16_t *>(to + 2 * nb) = (uint16_t)(code[4] | code[5] << 4 | code[6] << 8 | code[7] << 12);
    } else {
        *reinterpret_cast<uint32_t *>(tile + p * 16 * nb + j * 4 * nb + 4 * k.b) = word;
    }
    if (j == 0) *reinterpret_cast<__half *>(tile + kv4_codes(nb) + p * 2 * nb + 2 * k.b) = dh;
}

// A token for each blockIdx.x, its rows dealt out over blockIdx.y.
template <typename T, KpTurn TURN>
__global__ void __launch_bounds__(kKpThreads, 8) kv4_append_kernel(const __grid_constant__ Kv4AppendArgs a) {
    pdl_wait();
    const uint32_t seq = blockIdx.x / a.n_query, t = blockIdx.x - seq * a.n_query, at = blockIdx.y * kKpThreads + threadIdx.x,
                   step = gridDim.y * kKpThreads;
    uint32_t bad = 0;
    const int32_t pos = kp_position(a, seq, t, bad);
    if (pos < 0) {
        if (bad && at == 0) atomicOr(a.err, bad);
        return;
    }
    const uint64_t from = seq * a.q.seq + t * a.q.tok, to = seq * a.q_out.seq + t * a.q_out.tok;
    const uint32_t nq = a.n_head * (a.hd * sizeof(T) / 32), nkv = 2 * a.n_kv * kv4_blocks(a.hd) * 4;
    const uint32_t page = (uint32_t)a.pages[seq * a.pages_seq + ((uint32_t)pos >> a.page_log2)];
    KpQuery<T> q;
    for (uint32_t i = at; i < nq; i += step) {
        kp_query_load<T>(a, i, from, q);
        kp_query_store<T, TURN>(a, q, to, (uint32_t)pos);
    }
    if (page >= a.n_page) {
        if (at == 0) atomicOr(a.err, kKvBadPage);
        return;
    }
    KpBlock k;
    for (uint32_t i = at; i - threadIdx.x % 32 < nkv; i += step) {
        kp_block_load<T, TURN>(a, i, seq, t, i < nkv, k);
        kp_block_store<TURN>(a, k, i, page, (uint32_t)pos, i < nkv);
    }
}

struct Kv4ReadArgs {
    const uint8_t *cache;
    const int32_t *pages, *start, *len;  // len may be null
    void *k, *v;                         // [n_seq][n][n_kv][hd], contiguous
    uint64_t pages_seq;
    uint32_t type, n_seq, n, n_kv, hd, page_log2, n_page, max_pages;
    uint32_t *err;
};

// Four values of a position's key or value row per thread: (code - 8) * d, exact
// in fp32 and rounded once to the type; zeros where there is no position.
__global__ void __launch_bounds__(kKpThreads) kv4_read_kernel(const __grid_constant__ Kv4ReadArgs a) {
    pdl_wait();
    const uint32_t part = a.hd / 4, i = blockIdx.x * kKpThreads + threadIdx.x, e = i % part, row = i / part,
                   h = row % (2 * a.n_kv), tok = row / (2 * a.n_kv), seq = tok / a.n, t = tok % a.n, nb = kv4_blocks(a.hd);
    if (seq >= a.n_seq) return;
    const bool value = h >= a.n_kv;
    const uint32_t head = value ? h - a.n_kv : h, b = e / 8, j = e % 8;
    const int64_t pos = (int64_t)a.start[seq] + t;
    float4 y = {0.f, 0.f, 0.f, 0.f};
    if (pos >= 0 && pos < (int64_t)a.max_pages << a.page_log2 && (!a.len || pos < a.len[seq])) {
        const uint32_t page = (uint32_t)a.pages[seq * a.pages_seq + (uint32_t)(pos >> a.page_log2)];
        if (page < a.n_page) {
            const uint32_t in = (uint32_t)pos & ((1u << a.page_log2) - 1), p = in % kKvTile;
            const uint8_t *tile = a.cache + ((((uint64_t)page * a.n_kv + head) << (a.page_log2 - 4)) + in / kKvTile) * kv4_tile(nb) +
                                  (value ? kv4_codes(nb) + kv4_scales(nb) : 0);
            const float d = __half2float(*reinterpret_cast<const __half *>(tile + kv4_codes(nb) + p * 2 * nb + 2 * b));
            uint32_t q;  // codes at bits 0, 4, 8, 12
            if (value) {
                q = *reinterpret_cast<const uint16_t *>(tile + p * 16 * nb + (j ^ (p & 2 ? 4u : 0u)) * 2 * nb + 2 * b);
            } else {
                const uint32_t w = *reinterpret_cast<const uint32_t *>(tile + p * 16 * nb + (j / 2) * 4 * nb + 4 * b) >> (j & 1 ? 8 : 0);
                q = (w & 15) | (w >> 16 & 15) << 4 | (w >> 4 & 15) << 8 | (w >> 20 & 15) << 12;
            }
            y.x = ((int)(q & 15) - 8) * d;
            y.y = ((int)(q >> 4 & 15) - 8) * d;
            y.z = ((int)(q >> 8 & 15) - 8) * d;
            y.w = ((int)(q >> 12 & 15) - 8) * d;
        } else {
            atomicOr(a.err, kKvBadPage);
        }
    }
    kv4_store4(value ? a.v : a.k, ((uint64_t)tok * a.n_kv + head) * a.hd + 32 * b + 4 * j, a.type, y);
}

}  // namespace fwb
