// kv4_attn.cuh — attention over the paged cache of 4-bit keys and values.
//
//     out = sum_p exp(s_p - lse) v_p,  s_p = scale q.k_p,  lse = log sum_p exp(s_p)
//
// for every query row (token x query head of a KV head) over the positions
// that its token sees.  A key is k = d_b (code - 8) in blocks b of 32, so
//
//     s_p = scale sum_b d_kb (codes_pb . q_b),   out = sum_p (exp(s_p - m) d_vb) codes_p
//
// and the products run on the codes, which fp16 holds exactly; the scales
// multiply the 32-wide partial scores and the probabilities in fp32.
//
// Bound: DRAM (72 bytes per position, head and side at head_dim 128) for large
// batches, the ends of the launch for small ones; see the figures at the
// kernel.  Positions are the rows of the m16n8k16 products and query rows the
// columns: a group's few rows fill 8 columns, and an instruction multiplies
// 256 values of K or V, which is what unpacking them at the memory's rate
// leaves room for.  (tcgen05 would want them unpacked into shared memory.)
//
// Work: an item is (sequence, row tile, KV head); the items' tiles of 16
// positions stand in one line that is cut evenly over the CTAs, an item's ends
// counting as kKaCost tiles.  The eight warps of a CTA take an item's tiles in
// turn, each with a ring of its own that it fills by 16-byte copies, and join
// their results in shared memory at the item's end.  Where an item is cut, its
// parts go to the workspace and the CTA that arrives last adds them, in the
// order of the positions whichever arrives last.
#pragma once
#include "kv4_format.cuh"

namespace fwb {

constexpr int kKaWarps = 8, kKaThreads = 32 * kKaWarps, kKaStages = 4;
constexpr float kKaLazy = 7.f;  // log2 of how far a score may exceed its row's reference
constexpr float kKaHead = 256.f;  // largest product of a probability and a scale when references are exact

struct Kv4AttnArgs {
    const void *q;
    const uint8_t *cache;
    const int32_t *pages, *len, *n_new;
    void *out;
    float *lse;
    uint64_t q_seq, q_tok, q_head, pages_seq;  // strides in elements
    uint32_t type, n_seq, n_query, n_head, n_kv, gq, hd;
    uint32_t tpp_log2, n_page, max_pages;  // tiles of a page
    uint32_t rtiles, cost, least;          // row tiles; units of an item's ends; units worth a CTA
    float scale;
    float *po;        // [2 CTAs][rows][32 NB] parts of cut items
    float2 *pml;      // [2 CTAs][rows] their references and sums
    uint32_t *ticket; // [CTAs] zero between launches
    uint32_t *err;
};

__device__ __forceinline__ float ka_exp2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
__device__ __forceinline__ void ka_mma(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
// The 8x8 halves that a warp holds as rows, as columns.
__device__ __forceinline__ uint32_t ka_transpose(uint32_t x) {
    uint32_t y;
    asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
    return y;
}
// The codes less 8 of nibbles (0, 4), (1, 5), (2, 6), (3, 7) as pairs of
// halves: 0x6400 is 1024, whose last bit is worth 1 (16 for the upper nibble
// of a byte), so 1024 + q and 1024 + 16 q need only their mask, and each
// subtraction or fma is exact.
__device__ __forceinline__ void ka_codes(uint32_t w, uint32_t (&h)[4]) {
    const __half2 k1032 = __half2half2(__ushort_as_half(0x6408)), k16 = __half2half2(__ushort_as_half(0x2c00)),
                  k72 = __half2half2(__ushort_as_half(0xd480));
#pragma unroll
    for (int i = 0; i < 2; ++i, w >>= 8) {
        const uint32_t lo = (w & 0x000f000fu) | 0x64006400u, hi = (w & 0x00f000f0u) | 0x64006400u;
        const __half2 a = __hsub2(*reinterpret_cast<const __half2 *>(&lo), k1032),
                      b = __hfma2(*reinterpret_cast<const __half2 *>(&hi), k16, k72);
        h[2 * i] = *reinterpret_cast<const uint32_t *>(&a);
        h[2 * i + 1] = *reinterpret_cast<const uint32_t *>(&b);
    }
}

// NB 32-bit words, or the units of NB 16-bit parts.
template <int NB>
__device__ __forceinline__ void ka_words(const uint8_t *p, uint32_t (&w)[NB]) {
    if constexpr (NB == 4) {
        const uint4 v = *reinterpret_cast<const uint4 *>(p);
        w[0] = v.x; w[1] = v.y; w[2] = v.z; w[3] = v.w;
    } else if constexpr (NB == 2) {
        const uint2 v = *reinterpret_cast<const uint2 *>(p);
        w[0] = v.x; w[1] = v.y;
    } else {
#pragma unroll
        for (int i = 0; i < NB; ++i) w[i] = reinterpret_cast<const uint32_t *>(p)[i];
    }
}
template <int NB>
__device__ __forceinline__ void ka_halves(const uint8_t *p, uint32_t (&w)[(NB + 1) / 2]) {
    if constexpr (NB == 4) {
        const uint2 v = *reinterpret_cast<const uint2 *>(p);
        w[0] = v.x; w[1] = v.y;
    } else if constexpr (NB == 2) {
        w[0] = *reinterpret_cast<const uint32_t *>(p);
    } else {
        const uint16_t *h = reinterpret_cast<const uint16_t *>(p);
        w[0] = NB == 1 ? h[0] : h[0] | (uint32_t)h[1] << 16;
        if constexpr (NB == 3) w[1] = h[2];
    }
}

// What an item needs to know of its rows.
struct KaItem {
    uint32_t seq, rt, head;
    uint32_t tiles;       // that its last row sees
    int32_t limit;        // positions that its last row sees
    int32_t len, fresh;   // of its sequence
};

// Positions that row `row` of the sequence sees; -1 behind the new tokens.
__device__ __forceinline__ int32_t ka_limit(const Kv4AttnArgs &a, int32_t len, int32_t fresh, uint32_t row) {
    const int32_t t = (int32_t)(row / a.gq);
    return t < fresh ? max(0, len - (fresh - 1 - t)) : -1;
}
__device__ __forceinline__ void ka_lengths(const Kv4AttnArgs &a, uint32_t seq, int32_t &len, int32_t &fresh) {
    len = min(max(a.len[seq], 0), (int32_t)((a.max_pages << a.tpp_log2) * kKvTile));
    fresh = a.n_new ? min(max(a.n_new[seq], 0), (int32_t)a.n_query) : (int32_t)a.n_query;
}
// The tiles of row tile rt of a sequence; false where it has no row.
template <int ROWS>
__device__ __forceinline__ bool ka_tiles(const Kv4AttnArgs &a, uint32_t rt, int32_t len, int32_t fresh, int32_t &limit) {
    const int32_t t0 = (int32_t)(rt * ROWS / a.gq);
    if (t0 >= fresh) return false;
    const int32_t t1 = min((int32_t)(((uint64_t)rt * ROWS + ROWS - 1) / a.gq), fresh - 1);
    limit = max(0, len - (fresh - 1 - t1));
    return true;
}

template <int NB, int NT>
struct KaSmem {
    static constexpr uint32_t kRows = 8 * NT, kTile = kv4_tile(NB), kStride = 32 * NB + 4;
    static constexpr uint32_t kRing = kKaWarps * kKaStages * kTile, kJoin = kKaWarps * kRows * kStride * 4;
    static constexpr uint32_t kBytes = kRing > kJoin ? kRing : kJoin;
};

// One tile of 16 positions.  EDGE: some rows may not see all of them.
template <bool SPLIT, int NB, int NT, bool EDGE>
__device__ __forceinline__ void ka_tile(const uint8_t *tile, const uint32_t (&qh)[NT][NB][4], const uint32_t (&ql)[SPLIT ? NT : 1][NB][4],
                                        const float (&qs)[NT][2], const int32_t (&lim)[NT][2], int32_t pos0, int32_t limit,
                                        float (&o)[NT][NB][2][4], float (&m)[NT][2], float (&l)[NT][2], float &vref) {
    const uint32_t lane = threadIdx.x & 31, g = lane >> 2, c = lane & 3;
    const uint32_t p0 = (g >> 1) + 4 * (g & 1), p1 = p0 + 8;  // the positions of this lane's rows of the scores
    float s[NT][4];
#pragma unroll
    for (int n = 0; n < NT; ++n) s[n][0] = s[n][1] = s[n][2] = s[n][3] = 0.f;
    {
        uint32_t w0[NB], w1[NB], d0[(NB + 1) / 2], d1[(NB + 1) / 2];
        ka_words<NB>(tile + p0 * 16 * NB + c * 4 * NB, w0);
        ka_words<NB>(tile + p1 * 16 * NB + c * 4 * NB, w1);
        ka_halves<NB>(tile + kv4_codes(NB) + p0 * 2 * NB, d0);
        ka_halves<NB>(tile + kv4_codes(NB) + p1 * 2 * NB, d1);
#pragma unroll
        for (int b = 0; b < NB; ++b) {
            uint32_t x[4], y[4];
            ka_codes(w0[b], x);
            ka_codes(w1[b], y);
            const float2 e0 = kv4_unpack(d0[b / 2]), e1 = kv4_unpack(d1[b / 2]);
            const float k0 = b % 2 ? e0.y : e0.x, k1 = b % 2 ? e1.y : e1.x;
            const uint32_t a0[4] = {x[0], y[0], x[1], y[1]}, a1[4] = {x[2], y[2], x[3], y[3]};
#pragma unroll
            for (int n = 0; n < NT; ++n) {
                float acc[4] = {0.f, 0.f, 0.f, 0.f};
                if constexpr (SPLIT) {
                    ka_mma(acc, a0, ql[n][b][0], ql[n][b][1]);
                    ka_mma(acc, a1, ql[n][b][2], ql[n][b][3]);
                }
                ka_mma(acc, a0, qh[n][b][0], qh[n][b][1]);
                ka_mma(acc, a1, qh[n][b][2], qh[n][b][3]);
                s[n][0] = fmaf(k0, acc[0], s[n][0]);
                s[n][1] = fmaf(k0, acc[1], s[n][1]);
                s[n][2] = fmaf(k1, acc[2], s[n][2]);
                s[n][3] = fmaf(k1, acc[3], s[n][3]);
            }
        }
    }
    bool seen[NT][4];
    bool raise = false;
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            s[n][i] *= qs[n][i & 1];
            if constexpr (EDGE) {
                seen[n][i] = pos0 + (int32_t)(i < 2 ? p0 : p1) < lim[n][i & 1];
                if (!seen[n][i]) s[n][i] = -INFINITY;
            }
            raise |= s[n][i] > m[n][i & 1] + kKaLazy;
        }
    // References follow the scores only when one exceeds its own by 2^7: the
    // products below stay under 2^15, which fp16 holds.
    if (__any_sync(0xffffffffu, raise)) {
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
            for (int j = 0; j < 2; ++j) {
                float top = fmaxf(s[n][j], s[n][j + 2]);
                top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 4));
                top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 8));
                top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 16));
                if (top > m[n][j]) {
                    const float f = ka_exp2(m[n][j] - top);
                    m[n][j] = top;
                    l[n][j] *= f;
#pragma unroll
                    for (int b = 0; b < NB; ++b)
#pragma unroll
                        for (int t = 0; t < 2; ++t) {
                            o[n][b][t][j] *= f;
                            o[n][b][t][j + 2] *= f;
                        }
                }
            }
    }
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int j = 0; j < 2; ++j) {
            const float ref = m[n][j] == -INFINITY ? 0.f : m[n][j];  // nothing seen yet: every score is -inf
            s[n][j] = ka_exp2(s[n][j] - ref);
            s[n][j + 2] = ka_exp2(s[n][j + 2] - ref);
            l[n][j] += s[n][j] + s[n][j + 2];
        }
    const uint8_t *vt = tile + kv4_codes(NB) + kv4_scales(NB);
    // The values' scales relative to the largest so far (as a power of two).
    float v0[NB], v1[NB];
    {
        uint32_t d0[(NB + 1) / 2], d1[(NB + 1) / 2];
        ka_halves<NB>(vt + kv4_codes(NB) + p0 * 2 * NB, d0);
        ka_halves<NB>(vt + kv4_codes(NB) + p1 * 2 * NB, d1);
        float top = 0.f;
#pragma unroll
        for (int b = 0; b < NB; ++b) {
            const float2 e0 = kv4_unpack(d0[b / 2]), e1 = kv4_unpack(d1[b / 2]);
            v0[b] = b % 2 ? e0.y : e0.x;
            v1[b] = b % 2 ? e1.y : e1.x;
            if constexpr (EDGE) {  // past the last row's positions lies anything
                if (pos0 + (int32_t)p0 >= limit) v0[b] = 0.f;
                if (pos0 + (int32_t)p1 >= limit) v1[b] = 0.f;
            }
            top = fmaxf(top, fmaxf(fabsf(v0[b]), fabsf(v1[b])));
        }
        if (__any_sync(0xffffffffu, top > vref)) {
            const uint32_t bits = __reduce_max_sync(0xffffffffu, __float_as_uint(fminf(top, 65536.f)));
            const float now = fmaxf(vref, __uint_as_float((bits + 0x7fffffu) & 0xff800000u));
            const float f = vref * __uint_as_float((254u << 23) - __float_as_uint(now));  // of powers of two
            vref = now;
#pragma unroll
            for (int n = 0; n < NT; ++n)
#pragma unroll
                for (int b = 0; b < NB; ++b)
#pragma unroll
                    for (int t = 0; t < 2; ++t)
#pragma unroll
                        for (int i = 0; i < 4; ++i) o[n][b][t][i] *= f;
        }
        // kKaHead / vref
        const float inv = __uint_as_float(((254u + 8u) << 23) - __float_as_uint(vref));
#pragma unroll
        for (int b = 0; b < NB; ++b) {
            v0[b] *= inv;
            v1[b] *= inv;
        }
    }
    uint32_t u[4][(NB + 1) / 2];
#pragma unroll
    for (int j = 0; j < 4; ++j) ka_halves<NB>(vt + (c + 4 * j) * 16 * NB + (g ^ (c & 2 ? 4u : 0u)) * 2 * NB, u[j]);
#pragma unroll
    for (int b = 0; b < NB; ++b) {
        const uint32_t pick = b % 2 ? 0x7632u : 0x5410u;
        uint32_t x[4], y[4];
        ka_codes(__byte_perm(u[0][b / 2], u[1][b / 2], pick), x);
        ka_codes(__byte_perm(u[2][b / 2], u[3][b / 2], pick), y);
        const uint32_t a0[4] = {x[0], x[1], y[0], y[1]}, a1[4] = {x[2], x[3], y[2], y[3]};
#pragma unroll
        for (int n = 0; n < NT; ++n) {
            float w[4] = {s[n][0] * v0[b], s[n][1] * v0[b], s[n][2] * v1[b], s[n][3] * v1[b]};
            if constexpr (EDGE)
#pragma unroll
                for (int i = 0; i < 4; ++i)
                    if (!seen[n][i]) w[i] = 0.f;  // (its scale may be NaN)
            const uint32_t h0 = kv4_pack(w[0], w[1]), h1 = kv4_pack(w[2], w[3]);
            const uint32_t b0 = ka_transpose(h0), b1 = ka_transpose(h1);
            if constexpr (SPLIT) {
                // The rest of each product as a second half, and sums of 16
                // positions added in rounded fp32: the tensor cores' own
                // additions truncate.
                const float2 f0 = kv4_unpack(h0), f1 = kv4_unpack(h1);
                const uint32_t r0 = ka_transpose(kv4_pack(w[0] - f0.x, w[1] - f0.y)),
                               r1 = ka_transpose(kv4_pack(w[2] - f1.x, w[3] - f1.y));
                float t0[4] = {0.f, 0.f, 0.f, 0.f}, t1[4] = {0.f, 0.f, 0.f, 0.f};
                ka_mma(t0, a0, r0, r1);
                ka_mma(t1, a1, r0, r1);
                ka_mma(t0, a0, b0, b1);
                ka_mma(t1, a1, b0, b1);
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    o[n][b][0][i] += t0[i];
                    o[n][b][1][i] += t1[i];
                }
            } else {
                ka_mma(o[n][b][0], a0, b0, b1);
                ka_mma(o[n][b][1], a1, b0, b1);
            }
        }
    }
}

// SPLIT: fp32 calls, whose queries and weighted probabilities go through the
// products as two halves each.  NT: column tiles of 8 query rows.
template <bool SPLIT, int NB, int NT>
__global__ void __launch_bounds__(kKaThreads, NT == 1 ? 2 : 1) kv4_attn_kernel(const __grid_constant__ Kv4AttnArgs a) {
    using S = KaSmem<NB, NT>;
    constexpr uint32_t ROWS = S::kRows;
    extern __shared__ __align__(128) uint8_t ring[];
    __shared__ float2 sml[kKaWarps][ROWS];
    __shared__ float sref[kKaWarps];
    __shared__ float sw[kKaWarps][ROWS];   // weights of the warps' results
    __shared__ float2 srow[ROWS];          // an item's references and sums
    __shared__ uint32_t scan[kKaWarps + 1], sfind[3], slast;
    const uint32_t tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, c = lane & 3;
    pdl_wait();

    // --- this CTA's part of the line ---
    const uint32_t entries = a.n_seq * a.rtiles, per = (entries + kKaThreads - 1) / kKaThreads;
    auto units_of = [&](uint32_t e) -> uint32_t {
        int32_t len, fresh, limit;
        ka_lengths(a, e / a.rtiles, len, fresh);
        return ka_tiles<ROWS>(a, e % a.rtiles, len, fresh, limit) ? (uint32_t)(limit + kKvTile - 1) / kKvTile + a.cost : 0;
    };
    uint32_t mine = 0;
    for (uint32_t e = tid * per; e < min(entries, (tid + 1) * per); ++e) mine += units_of(e) * a.n_kv;
    uint32_t before = mine;
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
        const uint32_t x = __shfl_up_sync(0xffffffffu, before, d);
        if (lane >= (uint32_t)d) before += x;
    }
    if (lane == 31) scan[warp + 1] = before;
    if (tid == 0) scan[0] = 0;
    __syncthreads();
    uint32_t total = 0, base = 0;
#pragma unroll
    for (int w = 0; w < kKaWarps; ++w) {
        if (w == (int)warp) base = total;
        total += scan[w + 1];
    }
    before += base - mine;
    const uint32_t chunk = max((total + gridDim.x - 1) / gridDim.x, a.least);
    const uint64_t lo64 = (uint64_t)blockIdx.x * chunk;
    if (lo64 >= total) return;
    const uint32_t lo = (uint32_t)lo64, hi = min(total, lo + chunk);
    if (mine && before <= lo && lo < before + mine) {
        uint32_t at = before, e = tid * per, n;
        while (at + (n = units_of(e) * a.n_kv) <= lo) at += n, ++e;
        sfind[0] = e;
        sfind[1] = at;
        sfind[2] = (lo - at) / (n / a.n_kv);
    }
    __syncthreads();
    uint32_t entry = sfind[0], head = sfind[2], units = units_of(entry);
    uint32_t start = sfind[1] + head * units;  // of the item

    while (true) {
        const uint32_t seq = entry / a.rtiles, rt = entry % a.rtiles;
        int32_t len, fresh, limit = 0;
        ka_lengths(a, seq, len, fresh);
        ka_tiles<ROWS>(a, rt, len, fresh, limit);
        const uint32_t tiles = (uint32_t)(limit + kKvTile - 1) / kKvTile;
        const uint32_t from = min(max(lo, start) - start, tiles), to = min(min(hi, start + units) - start, tiles);
        if (from < to || (tiles == 0 && lo <= start)) {
            // --- queries: the products' B operand, columns of 8 rows ---
            uint32_t qh[NT][NB][4], ql[SPLIT ? NT : 1][NB][4];
            float qs[NT][2], m[NT][2], l[NT][2], o[NT][NB][2][4], vref = 5.9604645e-8f;  // 2^-24
            int32_t lim[NT][2];
            const uint32_t rows = a.n_query * a.gq;
#pragma unroll
            for (int n = 0; n < NT; ++n) {
                const uint32_t row = rt * ROWS + n * 8 + g, t = row / a.gq;
                float x[NB][8];
                float top = 0.f, odd = 0.f;
#pragma unroll
                for (int b = 0; b < NB; ++b) {
                    const uint32_t d = 32 * b + 8 * c;
                    float4 v0 = {0.f, 0.f, 0.f, 0.f}, v1 = v0;
                    if (row < rows && (int32_t)t < fresh && d < a.hd) {
                        const uint64_t at = seq * a.q_seq + t * a.q_tok + (head * a.gq + row % a.gq) * a.q_head + d;
                        v0 = kv4_load4(a.q, at, a.type);
                        v1 = kv4_load4(a.q, at + 4, a.type);
                    }
                    x[b][0] = v0.x; x[b][1] = v0.y; x[b][2] = v0.z; x[b][3] = v0.w;
                    x[b][4] = v1.x; x[b][5] = v1.y; x[b][6] = v1.z; x[b][7] = v1.w;
#pragma unroll
                    for (int i = 0; i < 8; ++i) {
                        top = fmaxf(top, fabsf(x[b][i]));
                        odd += x[b][i] * 0.f;  // NaN where something is not finite
                    }
                }
                top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
                top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
                odd += __shfl_xor_sync(0xffffffffu, odd, 1);
                odd += __shfl_xor_sync(0xffffffffu, odd, 2);
                // the row times a power of two, its largest value in [2^13, 2^14)
                const uint32_t ex = min(max(__float_as_uint(top) >> 23, 14u), 254u);
                const float up = __uint_as_float((267u - ex) << 23), down = __uint_as_float((ex - 13u) << 23) + odd;
#pragma unroll
                for (int b = 0; b < NB; ++b)
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        const float y0 = x[b][2 * i] * up, y1 = x[b][2 * i + 1] * up;
                        qh[n][b][i] = kv4_pack(y0, y1);
                        if constexpr (SPLIT) {
                            const float2 f = kv4_unpack(qh[n][b][i]);
                            ql[n][b][i] = kv4_pack(y0 - f.x, y1 - f.y);
                        }
                    }
#pragma unroll
                for (int j = 0; j < 2; ++j) {
                    qs[n][j] = __shfl_sync(0xffffffffu, down, 4 * (2 * c + j)) * (a.scale * 1.4426950408889634f);
                    lim[n][j] = ka_limit(a, len, fresh, rt * ROWS + n * 8 + 2 * c + j);
                    m[n][j] = -INFINITY;
                    l[n][j] = 0.f;
                }
#pragma unroll
                for (int b = 0; b < NB; ++b)
#pragma unroll
                    for (int i = 0; i < 4; ++i) o[n][b][0][i] = o[n][b][1][i] = 0.f;
            }
            const int32_t least = ka_limit(a, len, fresh, rt * ROWS);  // of the first row: the fewest positions

            // --- the warp's tiles ---
            uint8_t *const mine_ring = ring + warp * (kKaStages * S::kTile);
            const uint32_t count = from + warp < to ? (to - from - warp + kKaWarps - 1) / kKaWarps : 0;
            const int32_t *const table = a.pages + seq * a.pages_seq;
            uint32_t ids = 0, good = 0;
            auto fill = [&](uint32_t i) {
                if (i < count) {
                    if (i % 32 == 0)
                        ids = i + lane < count ? (uint32_t)table[(from + warp + (i + lane) * kKaWarps) >> a.tpp_log2] : 0;
                    const uint32_t page = __shfl_sync(0xffffffffu, ids, i % 32), stage = i % kKaStages;
                    good &= ~(1u << stage);
                    if (page < a.n_page) {
                        good |= 1u << stage;
                        const uint32_t t = from + warp + i * kKaWarps;
                        const uint8_t *src = a.cache + ((((uint64_t)page * a.n_kv + head) << a.tpp_log2) +
                                                        (t & ((1u << a.tpp_log2) - 1))) * S::kTile;
                        uint8_t *dst = mine_ring + stage * S::kTile;
                        constexpr uint32_t kChunks = S::kTile / 16;
#pragma unroll
                        for (uint32_t k = 0; k < (kChunks + 31) / 32; ++k)
                            if (k * 32 + lane < kChunks) cp_async16(dst + (k * 32 + lane) * 16, src + (k * 32 + lane) * 16);
                    } else if (lane == 0) {
                        atomicOr(a.err, kKvBadPage);
                    }
                }
                cp_async_commit();
            };
#pragma unroll
            for (uint32_t i = 0; i < kKaStages - 1; ++i) fill(i);
            for (uint32_t i = 0; i < count; ++i) {
                asm volatile("cp.async.wait_group %0;" ::"n"(kKaStages - 2) : "memory");
                __syncwarp();
                const uint32_t stage = i % kKaStages, t = from + warp + i * kKaWarps;
                if (good >> stage & 1) {
                    const uint8_t *tile = mine_ring + stage * S::kTile;
                    const int32_t pos0 = (int32_t)(t * kKvTile);
                    if (pos0 + (int32_t)kKvTile > least)
                        ka_tile<SPLIT, NB, NT, true>(tile, qh, ql, qs, lim, pos0, limit, o, m, l, vref);
                    else
                        ka_tile<SPLIT, NB, NT, false>(tile, qh, ql, qs, lim, pos0, limit, o, m, l, vref);
                }
                __syncwarp();
                fill(i + kKaStages - 1);
            }
            asm volatile("cp.async.wait_group 0;" ::: "memory");
            __syncthreads();  // the rings are free for the results

            // --- the warps' results joined ---
            float *const so = reinterpret_cast<float *>(ring);
#pragma unroll
            for (int n = 0; n < NT; ++n)
#pragma unroll
                for (int j = 0; j < 2; ++j) {
                    float sum = l[n][j];
                    sum += __shfl_xor_sync(0xffffffffu, sum, 4);
                    sum += __shfl_xor_sync(0xffffffffu, sum, 8);
                    sum += __shfl_xor_sync(0xffffffffu, sum, 16);
                    const uint32_t row = n * 8 + 2 * c + j;
                    if (g == 0) sml[warp][row] = make_float2(m[n][j], sum);
#pragma unroll
                    for (int b = 0; b < NB; ++b)
                        *reinterpret_cast<float4 *>(so + (warp * ROWS + row) * S::kStride + 32 * b + 4 * g) =
                            make_float4(o[n][b][0][j], o[n][b][0][j + 2], o[n][b][1][j], o[n][b][1][j + 2]);
                }
            if (lane == 0) sref[warp] = vref;
            __syncthreads();
            if (tid < ROWS) {
                float top = -INFINITY, sum = 0.f;
#pragma unroll
                for (int w = 0; w < kKaWarps; ++w) top = fmaxf(top, sml[w][tid].x);
                const float ref = top == -INFINITY ? 0.f : top;
#pragma unroll
                for (int w = 0; w < kKaWarps; ++w) {
                    const float f = ka_exp2(sml[w][tid].x - ref);
                    sum = fmaf(f, sml[w][tid].y, sum);
                    sw[w][tid] = f * sref[w] * (1.f / kKaHead);
                }
                srow[tid] = make_float2(top, sum);
            }
            __syncthreads();
            const uint32_t first = start / chunk, parts = (start + max(tiles, 1u) - 1) / chunk - first + 1;
            const bool begins = first == blockIdx.x;
            auto finish = [&](uint32_t r, uint32_t d, float4 v, float2 ml) {
                const uint32_t row = rt * ROWS + r, t = row / a.gq;
                if (row >= rows || (int32_t)t >= fresh) return;
                const uint64_t at = ((uint64_t)seq * a.n_query + t) * a.n_head + head * a.gq + row % a.gq;
                const float by = ml.y == 0.f ? 0.f : 1.f / ml.y;
                if (d < a.hd) kv4_store4(a.out, at * a.hd + d, a.type, make_float4(v.x * by, v.y * by, v.z * by, v.w * by));
                if (d == 0 && a.lse) a.lse[at] = ml.y == 0.f ? -INFINITY : (ml.x + log2f(ml.y)) * 0.69314718055994531f;
            };
            const uint64_t slot = 2ull * blockIdx.x + (begins ? 1 : 0);
            for (uint32_t i = tid; i < ROWS * 8 * NB; i += kKaThreads) {
                const uint32_t r = i / (8 * NB), d = i % (8 * NB) * 4;
                float4 v = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
                for (int w = 0; w < kKaWarps; ++w) {
                    const float4 x = *reinterpret_cast<const float4 *>(so + (w * ROWS + r) * S::kStride + d);
                    const float f = sw[w][r];
                    v.x = fmaf(f, x.x, v.x);
                    v.y = fmaf(f, x.y, v.y);
                    v.z = fmaf(f, x.z, v.z);
                    v.w = fmaf(f, x.w, v.w);
                }
                if (parts == 1) {
                    finish(r, d, v, srow[r]);
                } else {
                    *reinterpret_cast<float4 *>(a.po + (slot * ROWS + r) * (32 * NB) + d) = v;
                    if (d == 0) a.pml[slot * ROWS + r] = srow[r];
                }
            }
            if (parts > 1) {
                __threadfence();
                __syncthreads();
                if (tid == 0) slast = atomicAdd(a.ticket + first, 1u) == parts - 1;
                __syncthreads();
                if (slast) {
                    __threadfence();
                    if (tid == 0) a.ticket[first] = 0;
                    auto slot_of = [&](uint32_t p) { return 2ull * (first + p) + (p == 0 ? 1 : 0); };
                    for (uint32_t i = tid; i < ROWS * 8 * NB; i += kKaThreads) {
                        const uint32_t r = i / (8 * NB), d = i % (8 * NB) * 4;
                        float2 ml = {-INFINITY, 0.f};
                        float4 v = {0.f, 0.f, 0.f, 0.f};
#pragma unroll 4
                        for (uint32_t p = 0; p < parts; ++p) {
                            const float2 y = __ldcg(a.pml + slot_of(p) * ROWS + r);
                            const float4 x = __ldcg(reinterpret_cast<const float4 *>(a.po + (slot_of(p) * ROWS + r) * (32 * NB) + d));
                            const float top = fmaxf(ml.x, y.x), ref = top == -INFINITY ? 0.f : top;
                            const float f0 = ka_exp2(ml.x - ref), f1 = ka_exp2(y.x - ref);
                            ml = make_float2(top, ml.y * f0 + y.y * f1);
                            v.x = v.x * f0 + x.x * f1;
                            v.y = v.y * f0 + x.y * f1;
                            v.z = v.z * f0 + x.z * f1;
                            v.w = v.w * f0 + x.w * f1;
                        }
                        finish(r, d, v, ml);
                    }
                }
            }
            __syncthreads();  // the results are read: the rings may be filled again
        }
        // --- the next item ---
        start += units;
        if (start >= hi) break;
        if (++head == a.n_kv) {
            head = 0;
            do units = units_of(++entry);
            while (!units);
        }
    }
}

}  // namespace fwb
