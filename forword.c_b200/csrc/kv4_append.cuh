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
// Bound: DRAM for prompts, the launch for steps.  Eight lanes hold a block, four
// values each: its scale is three shuffles, and every store goes to bytes of
// this position alone.
#pragma once
#include "kv4_format.cuh"

namespace fwb {

constexpr int kKpThreads = 256;

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
    uint32_t type, n_seq, n_query, n_head, n_kv, hd, page_log2, n_page, max_pages, n_pos, halves;
    uint32_t q_blocks;  // CTAs for queries, before those for keys and values
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

// A rotated pair to fp32: in fp32 for queries (two roundings), exactly and
// then rounded for keys.
template <bool EXACT>
__device__ __forceinline__ float2 kp_turn(float x, float y, float c, float s) {
    if constexpr (EXACT)
        return make_float2((float)((double)x * c - (double)y * s), (float)((double)x * s + (double)y * c));
    else
        return make_float2(fmaf(x, c, -(y * s)), fmaf(x, s, y * c));
}

// Eight values of a query row: four pairs, so that a row may be turned in place.
__device__ __forceinline__ void kp_query(const Kv4AppendArgs &a, uint32_t i, uint32_t &bad) {
    const uint32_t part = a.hd / 8, j = i % part, row = i / part, h = row % a.n_head, tok = row / a.n_head,
                   seq = tok / a.n_query, t = tok % a.n_query;
    if (seq >= a.n_seq) return;
    const int32_t pos = kp_position(a, seq, t, bad);
    if (pos < 0) return;
    const uint32_t d0 = a.halves ? 4 * j : 8 * j, d1 = a.halves ? 4 * j + a.hd / 2 : 8 * j + 4;
    const uint64_t from = seq * a.q.seq + t * a.q.tok + h * a.q.head,
                   to = seq * a.q_out.seq + t * a.q_out.tok + h * a.q_out.head;
    float4 x = kv4_load4(a.q.p, from + d0, a.type), y = kv4_load4(a.q.p, from + d1, a.type);
    if (a.cos) {
        const uint64_t at = (uint64_t)pos * (a.hd / 2) + 4 * j;
        const float4 c = *reinterpret_cast<const float4 *>(a.cos + at), s = *reinterpret_cast<const float4 *>(a.sin + at);
        if (a.halves) {
            const float2 p0 = kp_turn<false>(x.x, y.x, c.x, s.x), p1 = kp_turn<false>(x.y, y.y, c.y, s.y),
                         p2 = kp_turn<false>(x.z, y.z, c.z, s.z), p3 = kp_turn<false>(x.w, y.w, c.w, s.w);
            x = make_float4(p0.x, p1.x, p2.x, p3.x);
            y = make_float4(p0.y, p1.y, p2.y, p3.y);
        } else {
            const float2 p0 = kp_turn<false>(x.x, x.y, c.x, s.x), p1 = kp_turn<false>(x.z, x.w, c.y, s.y),
                         p2 = kp_turn<false>(y.x, y.y, c.z, s.z), p3 = kp_turn<false>(y.z, y.w, c.w, s.w);
            x = make_float4(p0.x, p0.y, p1.x, p1.y);
            y = make_float4(p2.x, p2.y, p3.x, p3.y);
        }
    }
    kv4_store4(const_cast<void *>(a.q_out.p), to + d0, a.type, x);
    kv4_store4(const_cast<void *>(a.q_out.p), to + d1, a.type, y);
}

// The code of y: floor(y / d + 8.5) held to 0..15, by exact comparisons (a
// multiple of d / 2 up to 8.5 d is exact in fp32).
__device__ __forceinline__ uint32_t kp_code(float y, float d) {
    if (d == 0.f) return 8;
    const float a = fabsf(d), z = d < 0.f ? -y : y;
    float f = fminf(fmaxf(floorf(__fdiv_rn(z, a) + 8.5f), 0.f), 15.f);
    if (z < (f - 8.5f) * a) f -= 1.f;
    else if (z >= (f - 7.5f) * a) f += 1.f;
    return (uint32_t)fminf(fmaxf(f, 0.f), 15.f);
}

// A block of a key or value row, four values in each of eight lanes (all of a
// warp's lanes come here together).
__device__ __forceinline__ void kp_block(const Kv4AppendArgs &a, uint32_t i, uint32_t &bad) {
    const uint32_t nb = kv4_blocks(a.hd), j = i % 8, unit = i / 8, b = unit % nb, row = unit / nb,
                   h = row % (2 * a.n_kv), tok = row / (2 * a.n_kv), seq = tok / a.n_query, t = tok % a.n_query;
    const bool value = h >= a.n_kv;
    const uint32_t head = value ? h - a.n_kv : h, d0 = 32 * b + 4 * j;
    const int32_t pos = seq < a.n_seq ? kp_position(a, seq, t, bad) : -1;
    float y[4] = {0.f, 0.f, 0.f, 0.f};
    if (pos >= 0 && d0 < a.hd) {
        const Kv4Rows &src = value ? a.v : a.k;
        const uint64_t from = seq * src.seq + t * src.tok + head * src.head;
        const float4 x = kv4_load4(src.p, from + d0, a.type);
        y[0] = x.x; y[1] = x.y; y[2] = x.z; y[3] = x.w;
        if (!value && a.cos) {
            const uint64_t at = (uint64_t)pos * (a.hd / 2);
            if (a.halves) {
                const bool upper = d0 >= a.hd / 2;
                const uint32_t e = upper ? d0 - a.hd / 2 : d0;
                const float4 z = kv4_load4(src.p, from + (upper ? e : e + a.hd / 2), a.type);
                const float4 c = *reinterpret_cast<const float4 *>(a.cos + at + e), s = *reinterpret_cast<const float4 *>(a.sin + at + e);
                const float2 p0 = upper ? kp_turn<true>(z.x, x.x, c.x, s.x) : kp_turn<true>(x.x, z.x, c.x, s.x),
                             p1 = upper ? kp_turn<true>(z.y, x.y, c.y, s.y) : kp_turn<true>(x.y, z.y, c.y, s.y),
                             p2 = upper ? kp_turn<true>(z.z, x.z, c.z, s.z) : kp_turn<true>(x.z, z.z, c.z, s.z),
                             p3 = upper ? kp_turn<true>(z.w, x.w, c.w, s.w) : kp_turn<true>(x.w, z.w, c.w, s.w);
                y[0] = upper ? p0.y : p0.x; y[1] = upper ? p1.y : p1.x;
                y[2] = upper ? p2.y : p2.x; y[3] = upper ? p3.y : p3.x;
            } else {
                const float2 c = *reinterpret_cast<const float2 *>(a.cos + at + d0 / 2),
                             s = *reinterpret_cast<const float2 *>(a.sin + at + d0 / 2);
                const float2 p0 = kp_turn<true>(x.x, x.y, c.x, s.x), p1 = kp_turn<true>(x.z, x.w, c.y, s.y);
                y[0] = p0.x; y[1] = p0.y; y[2] = p1.x; y[3] = p1.y;
            }
        }
    }
    float hi = fmaxf(fmaxf(y[0], y[1]), fmaxf(y[2], y[3])), lo = fminf(fminf(y[0], y[1]), fminf(y[2], y[3]));
    uint32_t odd = !(fabsf(y[0]) < INFINITY && fabsf(y[1]) < INFINITY && fabsf(y[2]) < INFINITY && fabsf(y[3]) < INFINITY);
#pragma unroll
    for (int m = 1; m < 8; m <<= 1) {
        hi = fmaxf(hi, __shfl_xor_sync(0xffffffffu, hi, m));
        lo = fminf(lo, __shfl_xor_sync(0xffffffffu, lo, m));
        odd |= __shfl_xor_sync(0xffffffffu, odd, m);
    }
    // a block with a value that is not finite is NaN throughout; past what fp16
    // scales reach (|m| > 524032) values are held to the largest
    const __half dh = odd ? __ushort_as_half(0x7fff)
                          : __float2half_rn(fminf(fmaxf((hi >= -lo ? hi : lo) * -0.125f, -65504.f), 65504.f));
    const float d = odd ? 0.f : __half2float(dh);
    uint32_t code[4];
#pragma unroll
    for (int k = 0; k < 4; ++k) code[k] = kp_code(y[k], d);
    // lane j's half of key word c = j / 2: nibbles 0, 4, 1, 5 or 2, 6, 3, 7
    uint32_t word = code[0] | code[1] << 16 | code[2] << 4 | code[3] << 20;
    if (j & 1) word <<= 8;
    word |= __shfl_xor_sync(0xffffffffu, word, 1);
    if (pos < 0) return;
    const uint32_t page = (uint32_t)a.pages[seq * a.pages_seq + ((uint32_t)pos >> a.page_log2)];
    if (page >= a.n_page) {
        bad |= kKvBadPage;
        return;
    }
    const uint32_t in = (uint32_t)pos & ((1u << a.page_log2) - 1), p = in % kKvTile;
    uint8_t *tile = a.cache + ((((uint64_t)page * a.n_kv + head) << (a.page_log2 - 4)) + in / kKvTile) * kv4_tile(nb) +
                    (value ? kv4_codes(nb) + kv4_scales(nb) : 0);
    if (value)
        *reinterpret_cast<uint16_t *>(tile + p * 16 * nb + (j ^ (p & 2 ? 4u : 0u)) * 2 * nb + 2 * b) =
            (uint16_t)(code[0] | code[1] << 4 | code[2] << 8 | code[3] << 12);
    else if (!(j & 1))
        *reinterpret_cast<uint32_t *>(tile + p * 16 * nb + (j / 2) * 4 * nb + 4 * b) = word;
    if (j == 0) *reinterpret_cast<__half *>(tile + kv4_codes(nb) + p * 2 * nb + 2 * b) = dh;
}

__global__ void __launch_bounds__(kKpThreads) kv4_append_kernel(const __grid_constant__ Kv4AppendArgs a) {
    pdl_wait();
    uint32_t bad = 0;
    if (blockIdx.x < a.q_blocks)
        kp_query(a, blockIdx.x * kKpThreads + threadIdx.x, bad);
    else
        kp_block(a, (blockIdx.x - a.q_blocks) * kKpThreads + threadIdx.x, bad);
    if (bad) atomicOr(a.err, bad);
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
