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
#include <cuda.h>
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "beam_status.cuh"
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

__device__ __forceinline__ constexpr bool beam_is_bf16(__half) { return false; }
__device__ __forceinline__ constexpr bool beam_is_bf16(__nv_bfloat16) { return true; }

// A length read from the device, held to the positions that the cache has.
__device__ __forceinline__ uint32_t beam_len(const int32_t *len, uint32_t i, uint32_t cap) {
    if (!len) return cap;
    const int32_t n = len[i];
    return n < 0 ? 0u : min((uint32_t)n, cap);
}

// ---------------------------------------------------------------------------
// The split of the work.  A "part" is one group's prefix (rows: the query
// heads of one KV head of all its beams and new tokens) or one sequence's
// suffix; an item is a part, a KV head and a tile of rows.  Every item is a
// run of units of 16 positions; all items' U units stand in one line, and CTA c
// of C <= U takes units [c U / C, (c + 1) U / C).  So every CTA reads as many
// positions as any other, whatever the lengths are, and an item that several
// CTAs share leaves one partial result (sum, maximum, weighted values) per
// CTA.  An item's beginning and end cost time of their own: it stands in the
// line with `cost` units more in front, in which nothing is read.  A second
// kernel joins a row's partial results of prefix and suffix.
// ---------------------------------------------------------------------------
constexpr uint32_t kBaUnit = 16;      // positions
constexpr int kBaThreads = 128;       // four warps that compute
constexpr int kBaLoader = 32;         // and one that loads

struct BeamAttnPlan {
    float *po, *so;        // partial weighted values of prefix and suffix items: [slot][rows][HD]
    float2 *pml, *sml;     // their (maximum in units of log2, sum): [slot][rows]
    uint2 *pcta, *scta;    // (first, last) CTA of each item
    uint32_t prow, srow;   // rows of a prefix / suffix tile
    uint32_t ptiles, stiles;  // row tiles of a group / of a sequence
    uint32_t ctas;
    uint32_t part0, parts;  // the parts that a kernel takes: part0 .. parts - 1
    uint32_t cost;         // units that an item's own work is worth
    uint32_t by_gq, by_query;  // 2^32 / d rounded up, of row numbers below 2^16 (0: d = 1)
    uint32_t tma;          // bit 0: tensor maps of the prefix, 1: of the suffix
};

// Where a CTA stands in the line of units.
struct BeamCursor {
    uint32_t part;         // 0..n_group-1: prefixes, then the sequences
    uint32_t kvh, tile;
    uint32_t pos, len;     // the item's next position and its length
    uint32_t left;         // positions that this CTA still takes, counted in whole units
};

__device__ __forceinline__ uint32_t beam_part_len(const BeamAttnArgs &a, uint32_t part) {
    return part < a.n_group ? beam_len(a.plen, part, a.pcap) : beam_len(a.slen, part - a.n_group, a.scap);
}
__device__ __forceinline__ uint32_t beam_units(uint32_t len) { return (len + kBaUnit - 1) / kBaUnit; }

// Units of a part in the line.
__device__ __forceinline__ uint32_t beam_part_units(const BeamAttnArgs &a, const BeamAttnPlan &p, uint32_t part) {
    const uint32_t units = beam_units(beam_part_len(a, part));
    return units ? (units + p.cost) * a.n_kv * (part < a.n_group ? p.ptiles : p.stiles) : 0;
}

// The cursor of this CTA's first unit; false when it has none.  Every warp
// scans the parts' lengths for itself, so no barrier is waited for.
__device__ __forceinline__ bool beam_first(const BeamAttnArgs &a, const BeamAttnPlan &p, BeamCursor &c) {
    const uint32_t lane = threadIdx.x & 31, first = p.part0 + lane;
    uint32_t mine = first < p.parts ? beam_part_units(a, p, first) : 0, total = mine;  // of the first 32 parts
    for (uint32_t i = first + 32; i < p.parts; i += 32) total += beam_part_units(a, p, i);
    total = __reduce_add_sync(0xffffffffu, total);
    // with fewer units than CTAs the first ones take one each, so that the
    // CTAs of an item are neighbours
    const uint32_t ctas = min(total, p.ctas);
    if (blockIdx.x >= ctas) return false;
    const uint32_t per = total / ctas, more = total - per * ctas;  // the first `more` CTAs take one more
    uint32_t off = blockIdx.x * per + min(blockIdx.x, more);
    c.left = per + (blockIdx.x < more);
    for (uint32_t i0 = p.part0;; i0 += 32) {
        if (i0 != p.part0) mine = i0 + lane < p.parts ? beam_part_units(a, p, i0 + lane) : 0;
        uint32_t upto = mine;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const uint32_t v = __shfl_up_sync(0xffffffffu, upto, o);
            if (lane >= (uint32_t)o) upto += v;
        }
        const uint32_t hit = __ballot_sync(0xffffffffu, off < upto);
        if (hit) {
            const int at = __ffs(hit) - 1;
            c.part = i0 + at;
            off -= __shfl_sync(0xffffffffu, upto - mine, at);
            break;
        }
        off -= __shfl_sync(0xffffffffu, upto, 31);
        if (i0 + 32 >= p.parts) return false;  // lengths that changed under the call
    }
    c.len = beam_part_len(a, c.part);
    const uint32_t units = beam_units(c.len) + p.cost, tiles = c.part < a.n_group ? p.ptiles : p.stiles;
    if (c.len == 0) return false;            // likewise
    const uint32_t item = off / units;
    off -= item * units;
    c.kvh = item / tiles;
    c.tile = item - c.kvh * tiles;
    c.pos = off > p.cost ? (off - p.cost) * kBaUnit : 0;
    if (off < p.cost) c.left -= min(c.left, p.cost - off);
    return c.left != 0;
}

// To the item after the cursor's (its positions are used up, units are left).
__device__ __forceinline__ void beam_next_item(const BeamAttnArgs &a, const BeamAttnPlan &p, BeamCursor &c) {
    c.pos = 0;
    c.left -= min(c.left, p.cost);
    if (++c.tile < (c.part < a.n_group ? p.ptiles : p.stiles)) return;
    c.tile = 0;
    if (++c.kvh < a.n_kv) return;
    c.kvh = 0;
    do {
        if (++c.part >= p.parts) {  // lengths that changed under the call
            c.left = 0;
            return;
        }
        c.len = beam_part_len(a, c.part);
    } while (c.len == 0);
}

// --- matrix instructions of a warp --------------------------------------------
__device__ __forceinline__ void ldm_x4(uint32_t *r, uint32_t addr) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr));
}
__device__ __forceinline__ void ldm_x4_t(uint32_t *r, uint32_t addr) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr));
}
__device__ __forceinline__ void mma16(float *c, const uint32_t *a, uint32_t b0, uint32_t b1, __half) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void mma16(float *c, const uint32_t *a, uint32_t b0, uint32_t b1, __nv_bfloat16) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void mma8(float *c, const uint32_t *a, uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k8.row.col.f32.tf32.tf32.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
// x = hi + lo: hi rounded to tf32's 11 significant bits, lo the exact rest
// (12 bits and a sign; the product takes its first 11).  By integer addition:
// the conversion instruction has a quarter of its rate (4 beams over 30000
// positions 70 us with it, 61 without).
__device__ __forceinline__ void tf32_split(float x, uint32_t &hi, uint32_t &lo) {
    hi = (__float_as_uint(x) + 0x1000u) & 0xffffe000u;
    lo = __float_as_uint(x - __uint_as_float(hi));
}
__device__ __forceinline__ uint32_t pack2(float a, float b, __half) {
    const __half2 h = __floats2half2_rn(a, b);
    return *reinterpret_cast<const uint32_t *>(&h);
}
__device__ __forceinline__ uint32_t pack2(float a, float b, __nv_bfloat16) {
    const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
    return *reinterpret_cast<const uint32_t *>(&h);
}
__device__ __forceinline__ float exp2_fast(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
// 16 bytes global -> shared, or zeros (the source is not read then).
__device__ __forceinline__ void cp_async16_or_zero(uint32_t dst, const void *src, bool take) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(take ? 16 : 0) : "memory");
}
template <int N>
__device__ __forceinline__ void cp_async_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }

// Shared-memory tile: sub-tiles of 128 bytes of every row, [sub][row][128 B],
// the 16-byte chunk index xor-ed by the row's low three bits, as the copy
// engine's 128-byte swizzle does.  ldmatrix (8 rows of one chunk) and the fp32
// reads of V (2 chunks of the rows 2 t) touch all banks; the fp32 reads of K
// (4 chunks of 2 rows) take two rounds.
template <typename T, int HD>
struct BeamTile {
    static constexpr int kEs = sizeof(T), kChunks = HD * kEs / 16, kKeys = kEs == 2 ? 64 : 32;
    static constexpr int kSub = HD * kEs / 128;
    static constexpr uint32_t kBytes = kKeys * HD * kEs;  // of K; V the same
    static __device__ __forceinline__ uint32_t at(uint32_t row, uint32_t chunk) {
        return (chunk >> 3) * (kKeys * 128) + row * 128 + (((chunk ^ row) & 7) << 4);
    }
};

// Stages of tiles: fp32 has the query rows in shared memory too (their
// registers would be twice the 16-bit types'), and two stages leave room for
// three CTAs.
template <typename T>
constexpr int kBaStages = sizeof(T) == 2 ? 3 : 2;
// Behind them: fp32 query rows of the tile's row groups, and in the same place
// the outputs that warps sharing rows hand over at an item's end.
template <typename T, int HD, int RW>
constexpr uint32_t beam_attn_rows_smem() {  // (a row group: 16 rows in the tiles' chunk order)
    return sizeof(T) == 4 ? RW * 16 * HD * 4 : RW < 4 ? 2 * 16 * HD * 4 : 0;
}
constexpr uint32_t kBaTail = 2 * 3 * 8 + 2 * 16 * 8;  // barriers; maxima and sums that are handed over
template <typename T, int HD, int RWP, int RWS>
constexpr uint32_t beam_attn_smem() {
    constexpr uint32_t p = beam_attn_rows_smem<T, HD, RWP>(), s = beam_attn_rows_smem<T, HD, RWS>();
    return 2 * BeamTile<T, HD>::kBytes * kBaStages<T> + (p > s ? p : s) + kBaTail;
}

__device__ __forceinline__ void tma_load_4d(uint32_t dst, const CUtensorMap *map, int32_t x, int32_t y, int32_t z,
                                            int32_t u, uint64_t *bar) {
    asm volatile(
        "cp.async.bulk.tensor.4d.shared::cta.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4, %5}], [%6];"
        ::"r"(dst), "l"(map), "r"(x), "r"(y), "r"(z), "r"(u), "r"(smem_u32(bar)) : "memory");
}

// The caches as 4-D tensors [group or sequence][kv_head][position][dim],
// boxes of 16 positions (a unit) and 128 bytes, 128-byte swizzle, zeros past
// the dimensions; wk, wv: the prefix in boxes of a whole tile's positions.
struct BeamMaps {
    CUtensorMap pk, pv, sk, sv, wk, wv;
};

// n positions of a part into stage `st`, by the loading warp: units of 16
// positions that stand together by the copy engine (where the strides allow
// tensor maps), others -- a unit of a suffix whose slots differ -- row by row
// with 16-byte asynchronous copies.  The stage's barrier takes 32 arrivals.
template <typename T, int HD>
__device__ __forceinline__ void beam_load(const BeamAttnArgs &a, const BeamAttnPlan &p, const BeamMaps &maps,
                                          const BeamCursor &c, uint32_t n, uint32_t st, uint64_t *bar) {
    using Tl = BeamTile<T, HD>;
    constexpr int NU = Tl::kKeys / kBaUnit, CH = Tl::kChunks, RP = CH < 32 ? 32 / CH : 1;
    const uint32_t lane = threadIdx.x & 31, ks = st, vs = st + Tl::kBytes, units = (n + kBaUnit - 1) / kBaUnit;
    const bool pre = c.part < a.n_group;
    const uint32_t s = c.part - a.n_group;
    // the cache row's sequence, or group, of rows lane and lane + 32
    uint32_t seq[(Tl::kKeys + 31) / 32], single = pre ? p.tma & 1 ? 0xfu : 0u : p.tma & 2 ? 0xfu : 0u;
#pragma unroll
    for (int i = 0; i < (Tl::kKeys + 31) / 32; ++i) seq[i] = pre ? c.part : s;
    if (!pre && a.slots) {
        const uint32_t b0 = s / a.n_beam * a.n_beam;
        const int32_t *slots = a.slots + s * a.slot_seq + c.pos;
#pragma unroll
        for (int i = 0; i < (Tl::kKeys + 31) / 32; ++i) {
            const uint32_t row = lane + 32 * i;
            if (row < n) {
                const uint32_t from = (uint32_t)slots[row];
                if (from < a.n_beam) seq[i] = b0 + from;
            }
        }
#pragma unroll
        for (int u = 0; u < NU; ++u) {  // units whose rows differ
            const uint32_t row = (u & 1) * kBaUnit, v = seq[u / 2];
            const uint32_t lead = __shfl_sync(0xffffffffu, v, row);
            const uint32_t off = __ballot_sync(0xffffffffu, v != lead && lane + (u & ~1) * kBaUnit < n);
            if (off >> row & 0xffffu) single &= ~(1u << u);
        }
    }
    if (pre && single && units == NU) {  // a whole tile: one box per sub-tile
        if (lane == 0)
            asm volatile("mbarrier.expect_tx.relaxed.cta.shared::cta.b64 [%0], %1;" ::"r"(smem_u32(bar)), "r"(2 * Tl::kBytes) : "memory");
        __syncwarp();
        if (lane < 2 * Tl::kSub) {
            const uint32_t h = lane % Tl::kSub;
            const bool k = lane < Tl::kSub;
            tma_load_4d((k ? ks : vs) + h * (Tl::kKeys * 128), k ? &maps.wk : &maps.wv, (int32_t)(h * (128 / Tl::kEs)),
                        (int32_t)c.pos, (int32_t)c.kvh, (int32_t)c.part, bar);
        }
        mbar_arrive(bar);
        return;
    }
    uint32_t bytes = 0;
#pragma unroll
    for (int u = 0; u < NU; ++u)
        if (u < units && single >> u & 1) bytes += 2 * Tl::kSub * kBaUnit * 128;
    if (lane == 0 && bytes)
        asm volatile("mbarrier.expect_tx.relaxed.cta.shared::cta.b64 [%0], %1;" ::"r"(smem_u32(bar)), "r"(bytes) : "memory");
#pragma unroll 1
    for (uint32_t u = 0; u < units; ++u) {
        const uint32_t r0 = u * kBaUnit;
        if (single >> u & 1) {
            const uint32_t from = __shfl_sync(0xffffffffu, u < 2 ? seq[0] : seq[(Tl::kKeys + 31) / 32 - 1], r0 & 31);
            // one box per lane: K and V, each sub-tile
            if (lane < 2 * Tl::kSub) {
                const uint32_t h = lane % Tl::kSub, to = h * (Tl::kKeys * 128) + r0 * 128;
                const bool k = lane < Tl::kSub;
                tma_load_4d((k ? ks : vs) + to, pre ? k ? &maps.pk : &maps.pv : k ? &maps.sk : &maps.sv,
                            (int32_t)(h * (128 / Tl::kEs)), (int32_t)(c.pos + r0), (int32_t)c.kvh, (int32_t)from, bar);
            }
            continue;
        }
        const uint32_t ch = lane % CH;
        const bool held = ch * (16 / Tl::kEs) < a.hd;
        const size_t outer = pre ? a.p_group : a.s_seq, step = pre ? a.p_pos : a.s_pos;
        const size_t col = (pre ? c.kvh * a.p_head : c.kvh * a.s_head) + (held ? (size_t)ch * (16 / Tl::kEs) : 0);
        const T *kb = static_cast<const T *>(pre ? a.pk : a.sk) + col, *vb = static_cast<const T *>(pre ? a.pv : a.sv) + col;
#pragma unroll 4
        for (uint32_t i = 0; i < kBaUnit; i += RP) {
            const uint32_t row = r0 + i + lane / CH;
            const uint32_t from = __shfl_sync(0xffffffffu, u < 2 ? seq[0] : seq[(Tl::kKeys + 31) / 32 - 1], row & 31);
            if (row < n) {
                const size_t off = from * outer + (size_t)(c.pos + row) * step;
                cp_async16_or_zero(ks + Tl::at(row, ch), kb + off, held);
                cp_async16_or_zero(vs + Tl::at(row, ch), vb + off, held);
            }
        }
    }
    asm volatile("cp.async.mbarrier.arrive.noinc.shared::cta.b64 [%0];" ::"r"(smem_u32(bar)) : "memory");
}

// The online softmax of a warp's 16 rows: thread rows g and g + 8 (g = lane
// / 4).  Scores come in sc (raw products), leave as probabilities relative
// to the new maximum; returns the factors of the earlier sums.
template <int NB>
__device__ __forceinline__ void beam_softmax(float (*sc)[4], float sl2, float *m, float *l, float *al) {
#pragma unroll
    for (int h = 0; h < 2; ++h) {
        float mx = -INFINITY;
#pragma unroll
        for (int j = 0; j < NB; ++j) mx = fmaxf(mx, fmaxf(sc[j][2 * h], sc[j][2 * h + 1]));
        mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 1));
        mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 2));
        const float mn = fmaxf(m[h], mx * sl2), safe = mn == -INFINITY ? 0.f : mn;
        al[h] = exp2_fast(m[h] - safe);
        m[h] = mn;
        float sum = 0.f;
#pragma unroll
        for (int j = 0; j < NB; ++j)
#pragma unroll
            for (int e = 2 * h; e < 2 * h + 2; ++e) {
                sc[j][e] = exp2_fast(fmaf(sc[j][e], sl2, -safe));
                sum += sc[j][e];
            }
        l[h] = fmaf(l[h], al[h], sum);  // the lanes' shares are joined at the end
    }
}

// Rows of one warp: 16 query rows in registers, their output, maximum, sum.
template <typename T, int HD>
struct BeamRows {
    uint32_t q[sizeof(T) == 2 ? HD / 4 : 1];  // matrix operand A, 16-bit types (fp32: in shared memory)
    float o[HD / 8][4];
    float m[2], l[2];
    int32_t lim[2];                  // positions that rows g and g + 8 see (-1: no such row)
};

__device__ __forceinline__ uint32_t beam_div(uint32_t n, uint32_t by) { return by ? __umulhi(n, by) : n; }

// Query row r of an item (row = (beam * n_query + token) * gq + head of the
// group), and the positions that it sees.
template <typename T, int HD>
__device__ __forceinline__ const T *beam_q_row(const BeamAttnArgs &a, const BeamAttnPlan &p, const BeamCursor &c,
                                               uint32_t r, int32_t &lim) {
    lim = -1;
    const uint32_t rows = (c.part < a.n_group ? a.n_beam : 1) * a.n_query * a.gq;
    if (r >= rows) return nullptr;
    const uint32_t st = beam_div(r, p.by_gq), sb = beam_div(st, p.by_query);
    const uint32_t h = c.kvh * a.gq + r - st * a.gq, t = st - sb * a.n_query;
    uint32_t s = c.part - a.n_group;
    if (c.part < a.n_group) {
        s = c.part * a.n_beam + sb;
        lim = 0x7fffffff;
    } else {
        const uint32_t hidden = a.n_query - 1 - t;
        lim = c.len > hidden ? (int32_t)(c.len - hidden) : 0;
    }
    return static_cast<const T *>(a.q) + s * a.q_seq + t * a.q_tok + h * a.q_head;
}

// fp32 query row and chunk: quarter-warps read 4 chunks of 2 rows.
template <int HD>
__device__ __forceinline__ uint32_t beam_q_at(uint32_t row, uint32_t chunk) {
    return (row * (HD / 4) + (chunk ^ ((row & 1) << 2))) * 16;
}

template <typename T, int HD>
__device__ __forceinline__ void beam_rows_init(const BeamAttnArgs &a, const BeamAttnPlan &p, const BeamCursor &c,
                                               uint32_t r0, uint32_t qs, BeamRows<T, HD> &w) {
    const uint32_t lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
    const T *q[2];
    q[0] = beam_q_row<T, HD>(a, p, c, r0 + g, w.lim[0]);
    q[1] = beam_q_row<T, HD>(a, p, c, r0 + g + 8, w.lim[1]);
    if constexpr (sizeof(T) == 2) {
#pragma unroll
        for (int k = 0; k < HD / 16; ++k)
#pragma unroll
            for (int e = 0; e < 4; ++e) {  // a0: (g, 2t), a1: (g + 8, 2t), a2: (g, 2t + 8), a3: (g + 8, 2t + 8)
                const uint32_t d = 16 * k + 2 * t + (e >= 2 ? 8 : 0);
                const T *p = q[e & 1];
                w.q[4 * k + e] = p && d < a.hd ? *reinterpret_cast<const uint32_t *>(p + d) : 0u;
            }
    } else {
        // Warps that share rows write the same values to the same places, and
        // each lane reads back only what it wrote.
#pragma unroll
        for (int k = 0; k < HD / 16; ++k)
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                const uint32_t d = 16 * k + 4 * t;
                float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
                if (q[e] && d < a.hd) v = *reinterpret_cast<const float4 *>(q[e] + d);
                asm volatile("st.shared.v4.f32 [%0], {%1,%2,%3,%4};" ::"r"(qs + beam_q_at<HD>(g + 8 * e, 4 * k + t)),
                             "f"(v.x), "f"(v.y), "f"(v.z), "f"(v.w) : "memory");
            }
    }
#pragma unroll
    for (int j = 0; j < HD / 8; ++j)
#pragma unroll
        for (int e = 0; e < 4; ++e) w.o[j][e] = 0.f;
    w.m[0] = w.m[1] = -INFINITY;
    w.l[0] = w.l[1] = 0.f;
}

// One tile: KW positions of it, from row k0 on, for this warp's 16 rows.
// `at`: the part's position of the tile's first row; `end`: the first
// position past the tile.
template <typename T, int HD, int KW>
__device__ __forceinline__ void beam_tile(BeamRows<T, HD> &w, uint32_t qs, uint32_t ks, uint32_t vs, uint32_t k0,
                                          uint32_t at, uint32_t end, float sl2) {
    using Tl = BeamTile<T, HD>;
    const uint32_t lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
    float sc[KW / 8][4];
#pragma unroll
    for (int j = 0; j < KW / 8; ++j)
#pragma unroll
        for (int e = 0; e < 4; ++e) sc[j][e] = 0.f;
    if constexpr (sizeof(T) == 2) {
#pragma unroll
        for (int k = 0; k < HD / 16; ++k)
#pragma unroll
            for (int j = 0; j < KW / 16; ++j) {
                uint32_t b[4];
                ldm_x4(b, ks + Tl::at(k0 + 16 * j + (lane & 7) + ((lane >> 4) << 3), 2 * k + ((lane >> 3) & 1)));
                mma16(sc[2 * j], w.q + 4 * k, b[0], b[1], T{});
                mma16(sc[2 * j + 1], w.q + 4 * k, b[2], b[3], T{});
            }
    } else {
        // The 16 dimensions 16 k ..: lane t takes 4 t .. 4 t + 3, the first two as
        // columns t and t + 4 of one product and the others of the next.  The
        // tensor cores' fp32 sums truncate: the large products are summed from
        // zero over 16 dimensions and added with one rounded addition; the
        // small ones, 2^-11 of them, have sums of their own.
        float lq[KW / 8][4], lk[KW / 8][4];
#pragma unroll
        for (int j = 0; j < KW / 8; ++j)
#pragma unroll
            for (int e = 0; e < 4; ++e) lq[j][e] = lk[j][e] = 0.f;
#pragma unroll
        for (int k = 0; k < HD / 16; ++k) {
            uint32_t ah[8], al[8];
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                float4 v;
                const uint32_t ad = qs + beam_q_at<HD>(g + 8 * e, 4 * k + t);
                asm volatile("ld.shared.v4.f32 {%0,%1,%2,%3}, [%4];" : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w) : "r"(ad));
                tf32_split(v.x, ah[e], al[e]);
                tf32_split(v.y, ah[2 + e], al[2 + e]);
                tf32_split(v.z, ah[4 + e], al[4 + e]);
                tf32_split(v.w, ah[6 + e], al[6 + e]);
            }
#pragma unroll
            for (int j = 0; j < KW / 8; ++j) {
                float4 v;
                const uint32_t ad = ks + Tl::at(k0 + 8 * j + g, 4 * k + t);
                asm volatile("ld.shared.v4.f32 {%0,%1,%2,%3}, [%4];" : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w) : "r"(ad));
                uint32_t bh[4], bl[4];
                tf32_split(v.x, bh[0], bl[0]);
                tf32_split(v.y, bh[1], bl[1]);
                tf32_split(v.z, bh[2], bl[2]);
                tf32_split(v.w, bh[3], bl[3]);
                float acc[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
                for (int s = 0; s < 2; ++s) {
                    mma8(lq[j], al + 4 * s, bh[2 * s], bh[2 * s + 1]);
                    mma8(lk[j], ah + 4 * s, bl[2 * s], bl[2 * s + 1]);
                    mma8(acc, ah + 4 * s, bh[2 * s], bh[2 * s + 1]);
                }
#pragma unroll
                for (int e = 0; e < 4; ++e) sc[j][e] += acc[e];
            }
        }
#pragma unroll
        for (int j = 0; j < KW / 8; ++j)
#pragma unroll
            for (int e = 0; e < 4; ++e) sc[j][e] += lq[j][e] + lk[j][e];
    }
    // positions that a row does not see
    const uint32_t first = at + k0, lim0 = min((uint32_t)w.lim[0], end), lim1 = min((uint32_t)w.lim[1], end);
    if (first + KW > min(lim0, lim1)) {
#pragma unroll
        for (int j = 0; j < KW / 8; ++j)
#pragma unroll
            for (int e = 0; e < 4; ++e)
                if (first + 8 * j + 2 * t + (e & 1) >= (e < 2 ? lim0 : lim1)) sc[j][e] = -INFINITY;
    }
    float al[2];
    beam_softmax<KW / 8>(sc, sl2, w.m, w.l, al);
    if (first + KW > end) {
        // V rows past the end: their probabilities are zero, and zero times
        // whatever the memory holds must be zero.  (The warps that share these
        // rows write the same zeros.)
        for (uint32_t i = lane; i < KW * Tl::kChunks; i += 32) {
            const uint32_t row = i / Tl::kChunks;
            if (first + row >= end)
                asm volatile("st.shared.v4.u32 [%0], {%1,%1,%1,%1};" ::"r"(vs + Tl::at(k0 + row, i % Tl::kChunks)), "r"(0) : "memory");
        }
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");  // before the copy engine writes there again
        __syncwarp();
    }
    if constexpr (sizeof(T) == 2) {
        if (__any_sync(0xffffffffu, al[0] != 1.f || al[1] != 1.f)) {  // rare once the maxima are found
#pragma unroll
            for (int j = 0; j < HD / 8; ++j) {
                w.o[j][0] *= al[0];
                w.o[j][1] *= al[0];
                w.o[j][2] *= al[1];
                w.o[j][3] *= al[1];
            }
        }
        // The products with V take the probabilities in V's type.  What that costs,
        // besides the output's own rounding, error against 64 bits of a result
        // rounded once / of this: fp16 2.1e-4 / 2.4e-4, bf16 1.7e-3 / 2.3e-3.
        // Carrying the rest of the probabilities in a second product would double
        // the work with V; the sums, maxima and the output so far are fp32.
#pragma unroll
        for (int k = 0; k < KW / 16; ++k) {
            uint32_t p[4];
            p[0] = pack2(sc[2 * k][0], sc[2 * k][1], T{});
            p[1] = pack2(sc[2 * k][2], sc[2 * k][3], T{});
            p[2] = pack2(sc[2 * k + 1][0], sc[2 * k + 1][1], T{});
            p[3] = pack2(sc[2 * k + 1][2], sc[2 * k + 1][3], T{});
#pragma unroll
            for (int j = 0; j < HD / 16; ++j) {
                uint32_t b[4];
                ldm_x4_t(b, vs + Tl::at(k0 + 16 * k + (lane & 7) + ((lane >> 3) & 1) * 8, 2 * j + (lane >> 4)));
                mma16(w.o[2 * j], p, b[0], b[1], T{});
                mma16(w.o[2 * j + 1], p, b[2], b[3], T{});
            }
        }
    } else {
        // Again from zero for each tile, added to the output with one rounded
        // fma that does the rescaling too.
        uint32_t ph[KW / 8][4], pl[KW / 8][4];  // columns t, t + 4: positions 2 t, 2 t + 1
#pragma unroll
        for (int k = 0; k < KW / 8; ++k) {
            tf32_split(sc[k][0], ph[k][0], pl[k][0]);
            tf32_split(sc[k][2], ph[k][1], pl[k][1]);
            tf32_split(sc[k][1], ph[k][2], pl[k][2]);
            tf32_split(sc[k][3], ph[k][3], pl[k][3]);
        }
#pragma unroll
        for (int j = 0; j < HD / 32; ++j) {
            float acc[4][4];
#pragma unroll
            for (int i = 0; i < 4; ++i)
#pragma unroll
                for (int e = 0; e < 4; ++e) acc[i][e] = 0.f;
#pragma unroll
            for (int k = 0; k < KW / 8; ++k) {
                float v[2][4];
#pragma unroll
                for (int r = 0; r < 2; ++r) {
                    const uint32_t ad = vs + Tl::at(k0 + 8 * k + 2 * t + r, 8 * j + g);
                    asm volatile("ld.shared.v4.f32 {%0,%1,%2,%3}, [%4];"
                                 : "=f"(v[r][0]), "=f"(v[r][1]), "=f"(v[r][2]), "=f"(v[r][3]) : "r"(ad));
                }
#pragma unroll
                for (int i = 0; i < 4; ++i) {  // column g of product i: dimension 32 j + 4 g + i
                    uint32_t h0, l0, h1, l1;
                    tf32_split(v[0][i], h0, l0);
                    tf32_split(v[1][i], h1, l1);
                    mma8(acc[i], pl[k], h0, h1);
                    mma8(acc[i], ph[k], l0, l1);
                    mma8(acc[i], ph[k], h0, h1);
                }
            }
#pragma unroll
            for (int i = 0; i < 4; ++i)
#pragma unroll
                for (int e = 0; e < 4; ++e) w.o[4 * j + i][e] = fmaf(w.o[4 * j + i][e], al[e >> 1], acc[i][e]);
        }
    }
}

// Joins the rows of the warps that share them -- the upper half of those that
// had positions hands over to the lower, in 16-bit types; in fp32, where there
// is room for one, one after the other hands over to the first -- which then
// writes the item's partial result.  buf: outputs of two warps (fp32: one for
// every row group).  busy: warps that share rows and had positions.  wild: the
// sign bit if values were left out for the joining kernel, which reads it
// from the sums.
template <typename T, int HD, int RW>
__device__ __forceinline__ void beam_flush(const BeamAttnArgs &a, const BeamAttnPlan &p, const BeamCursor &c,
                                           BeamRows<T, HD> &w, uint32_t busy, uint32_t wild, float *buf, float2 *bml) {
    const uint32_t lane = threadIdx.x & 31, warp = threadIdx.x >> 5, rg = warp % RW, kg = warp / RW;
    const uint32_t g = lane >> 2, t = lane & 3;
#pragma unroll
    for (int h = 0; h < 2; ++h) {
        w.l[h] += __shfl_xor_sync(0xffffffffu, w.l[h], 1);
        w.l[h] += __shfl_xor_sync(0xffffffffu, w.l[h], 2);
    }
    constexpr bool kPairs = sizeof(T) == 2 && RW == 1;  // two hand over at once
#pragma unroll 1
    for (uint32_t i = 1; i < (kPairs ? 3u : 4u / RW); ++i) {
        const uint32_t half = kPairs ? 4 >> i : 1, from = kPairs ? half : i;
        if (from >= busy) continue;
        const uint32_t at = kPairs ? kg & (half - 1) : rg;
        float *ob = buf + at * 16 * HD;
        bar_sync(1, kBaThreads);  // what was here is read
        if (kg >= from && kg < from + half) {
#pragma unroll
            for (int j = 0; j < HD / 8; ++j)
                *reinterpret_cast<float4 *>(ob + (j * 32 + lane) * 4) =
                    make_float4(w.o[j][0], w.o[j][1], w.o[j][2], w.o[j][3]);
            if (t == 0) {
                bml[at * 16 + g] = make_float2(w.m[0], w.l[0]);
                bml[at * 16 + g + 8] = make_float2(w.m[1], w.l[1]);
            }
        }
        bar_sync(1, kBaThreads);
        if (kg < half) {
            float mine[2], other[2];
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                const float2 ml = bml[at * 16 + g + 8 * h];
                const float mn = fmaxf(w.m[h], ml.x), safe = mn == -INFINITY ? 0.f : mn;
                mine[h] = exp2_fast(w.m[h] - safe);
                other[h] = exp2_fast(ml.x - safe);
                w.m[h] = mn;
                w.l[h] = w.l[h] * mine[h] + ml.y * other[h];
            }
#pragma unroll
            for (int j = 0; j < HD / 8; ++j) {
                const float4 v = *reinterpret_cast<const float4 *>(ob + (j * 32 + lane) * 4);
                w.o[j][0] = w.o[j][0] * mine[0] + v.x * other[0];
                w.o[j][1] = w.o[j][1] * mine[0] + v.y * other[0];
                w.o[j][2] = w.o[j][2] * mine[1] + v.z * other[1];
                w.o[j][3] = w.o[j][3] * mine[1] + v.w * other[1];
            }
        }
    }
    // before the next item's rows come into the same place: these outputs', and
    // fp32 query rows of other warps where a suffix tile has fewer row groups
    if (RW < 4 || sizeof(T) == 4) bar_sync(1, kBaThreads);
    if (kg == 0) {
        const bool pre = c.part < a.n_group;
        const uint32_t item = ((pre ? c.part : c.part - a.n_group) * a.n_kv + c.kvh) * (pre ? p.ptiles : p.stiles) + c.tile;
        const size_t row = (size_t)(item + blockIdx.x) * (pre ? p.prow : p.srow) + rg * 16;
        float *o = (pre ? p.po : p.so) + row * HD;
        float2 *ml = (pre ? p.pml : p.sml) + row;
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            if (w.lim[h] < 0) continue;  // no such row
            float *r = o + (size_t)(g + 8 * h) * HD;
            if constexpr (sizeof(T) == 2) {
#pragma unroll
                for (int j = 0; j < HD / 8; ++j)
                    *reinterpret_cast<float2 *>(r + 8 * j + 2 * t) = make_float2(w.o[j][2 * h], w.o[j][2 * h + 1]);
            } else {
#pragma unroll
                for (int j = 0; j < HD / 32; ++j)
#pragma unroll
                    for (int e = 0; e < 2; ++e)
                        *reinterpret_cast<float4 *>(r + 32 * j + 8 * t + 4 * e) =
                            make_float4(w.o[4 * j][2 * h + e], w.o[4 * j + 1][2 * h + e], w.o[4 * j + 2][2 * h + e],
                                        w.o[4 * j + 3][2 * h + e]);
            }
            if (t == 0) ml[g + 8 * h] = make_float2(w.m[h], __uint_as_float(__float_as_uint(w.l[h]) | wild));
        }
    }
}

// The positions of the cursor's next tile: within the item and this CTA's units.
template <typename T, int HD>
__device__ __forceinline__ uint32_t beam_take(const BeamCursor &c) {
    return min(min((uint32_t)BeamTile<T, HD>::kKeys, c.len - c.pos), min(c.left, 4u) * kBaUnit);
}
__device__ __forceinline__ void beam_advance(BeamCursor &c, uint32_t n) {
    c.pos += n;
    c.left -= (n + kBaUnit - 1) / kBaUnit;
}

// Which halves of a word of V (fp32: whether it) are infinite or NaN, as bits
// 15 and 31 (31).
template <typename T> __device__ __forceinline__ uint32_t beam_wild(uint32_t x) {
    if constexpr (sizeof(T) == 4) return ((x & 0x7f800000u) + 0x00800000u) & 0x80000000u;
    else if constexpr (std::is_same<T, __half>::value) return ((x & 0x7c007c00u) + 0x04000400u) & 0x80008000u;
    else return ((x & 0x7f807f80u) + 0x00800080u) & 0x80008000u;
}

// A tile of which rows see different positions (several new tokens): a value
// of V that is infinite or NaN must not meet the zero probability of a row
// that does not see it.  It is made zero here, and the joining kernel adds it
// to the rows that do see it; rare, so it looks for it in the cache again.
// All computing threads, on the tile's first n positions.  Returns the sign
// bit where there was one.  Measured: 9 bf16 beams of 7 tokens, 71 suffix
// positions each, 30.8 us with the look and 30.1 without.
template <typename T, int HD>
__device__ __forceinline__ uint32_t beam_tame(uint32_t vs, uint32_t n) {
    using Tl = BeamTile<T, HD>;
    auto load = [&](uint32_t i, uint32_t *x) {
        const uint32_t ad = vs + Tl::at(i / Tl::kChunks, i % Tl::kChunks);
        asm volatile("ld.shared.v4.u32 {%0,%1,%2,%3}, [%4];" : "=r"(x[0]), "=r"(x[1]), "=r"(x[2]), "=r"(x[3]) : "r"(ad));
        return ad;
    };
    uint32_t x[4], wild = 0;
    for (uint32_t i = threadIdx.x; i < n * Tl::kChunks; i += kBaThreads) {
        load(i, x);
        wild |= beam_wild<T>(x[0]) | beam_wild<T>(x[1]) | beam_wild<T>(x[2]) | beam_wild<T>(x[3]);
    }
    asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.u32 p, %0, 0;\n\tbarrier.cta.red.or.pred p, 1, %1, p;\n\t"
                 "selp.u32 %0, 0x80000000, 0, p;\n\t}" : "+r"(wild) : "r"((uint32_t)kBaThreads) : "memory");
    if (!wild) return 0;
    for (uint32_t i = threadIdx.x; i < n * Tl::kChunks; i += kBaThreads) {
        const uint32_t ad = load(i, x);
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            const uint32_t b = beam_wild<T>(x[k]);
            x[k] = sizeof(T) == 4 ? (b ? 0u : x[k]) : x[k] & ~((b >> 15) * 0xffffu);
        }
        asm volatile("st.shared.v4.u32 [%0], {%1,%2,%3,%4};" ::"r"(ad), "r"(x[0]), "r"(x[1]), "r"(x[2]), "r"(x[3]) : "memory");
    }
    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");  // before the copy engine writes there again
    bar_sync(1, kBaThreads);
    return wild;
}

// One tile of the cursor's item: the item's first of this CTA brings in its
// query rows, the last writes the partial result.  RW warps hold the row
// groups of 16, and 4 / RW warps share each tile's positions.
template <typename T, int HD, int RW>
__device__ __forceinline__ void beam_step(const BeamAttnArgs &a, const BeamAttnPlan &p, BeamCursor &c, bool &fresh,
                                          uint32_t &most, uint32_t &wild, BeamRows<T, HD> &w, uint32_t stage, uint64_t *full, uint64_t *empty,
                                          uint32_t phase, bool &ok, uint32_t rows, float *buf, float2 *bml) {
    using Tl = BeamTile<T, HD>;
    constexpr int KW = Tl::kKeys / (4 / RW);
    const uint32_t warp = threadIdx.x >> 5, rg = warp % RW, kg = warp / RW;
    const uint32_t qs = rows + rg * 16 * HD * 4;
    if (fresh) {
        beam_rows_init<T, HD>(a, p, c, c.tile * RW * 16 + rg * 16, qs, w);
        most = wild = 0;
    }
    const bool first = c.pos == 0;
    const uint32_t n = beam_take<T, HD>(c);
    most = max(most, n);  // positions of the item's longest tile here
    // (after a wait that ran out: the same steps and barriers without the work)
    ok = mbar_wait_warp(full, phase, &g_beam_err, ERR_WAIT_FULL) && ok;
    if (c.part >= a.n_group && c.pos + n + a.n_query > c.len + 1) wild |= beam_tame<T, HD>(stage + Tl::kBytes, n);
    if (ok && kg * KW < n && __any_sync(0xffffffffu, w.lim[0] >= 0 || w.lim[1] >= 0))
        beam_tile<T, HD, KW>(w, qs, stage, stage + Tl::kBytes, kg * KW, c.pos, c.pos + n, a.scale * 1.4426950408889634f);
    __syncwarp();
    if ((threadIdx.x & 31) == 0) mbar_arrive(empty);
    beam_advance(c, n);
    fresh = c.pos >= c.len || c.left == 0;
    if (fresh) beam_flush<T, HD, RW>(a, p, c, w, (most + KW - 1) / KW, wild, buf, bml);
    if (threadIdx.x == 0 && (first || c.pos >= c.len)) {
        const bool pre = c.part < a.n_group;
        const uint32_t item = ((pre ? c.part : c.part - a.n_group) * a.n_kv + c.kvh) * (pre ? p.ptiles : p.stiles) + c.tile;
        uint2 *cta = (pre ? p.pcta : p.scta) + item;
        if (first) cta->x = blockIdx.x;
        if (c.pos >= c.len) cta->y = blockIdx.x;
    }
    if (fresh && c.left) beam_next_item(a, p, c);
}

// The attention of all parts, or of the suffixes alone.  RWP, RWS: row groups
// of 16 of a prefix / suffix tile.
//
// Bound: K and V once from DRAM.  Why this shape: 16 rows and 128 dimensions
// of output are 64 registers a lane, so a warp holds one row group and warps
// share positions when the rows are few (each K/V element is then read from
// shared memory once); two CTAs of a loading and four computing warps fill
// registers and shared memory (three for fp32 with 16 rows, whose query rows
// are in shared memory).  A tile of 32 KB takes a warp about 1200 (one row
// group) to 3500 cycles (four, fp16), 4000 in fp32.  Measured, whole calls on
// the device, without the host's part:
// fp16, 8 KV heads of 128, 30000 positions: 16 rows 30 us (4.1 TB/s), 32 rows
// 32, 64 rows 47; fp32, 8000 positions, 16 rows 26 us (2.6 TB/s); 9 us for
// 500 positions, which is what a call costs at least.
template <typename T, int HD, int RWP, int RWS>
__global__ void __launch_bounds__(kBaThreads + kBaLoader, sizeof(T) == 4 && RWP == 1 ? 3 : 2)
    beam_attn_kernel(const BeamAttnArgs a, const BeamAttnPlan p, const __grid_constant__ BeamMaps maps) {
    using Tl = BeamTile<T, HD>;
    constexpr int S = kBaStages<T>;
    // (the 128-byte swizzle counts rows from 1024-byte boundaries; nothing
    // static stands before this)
    extern __shared__ __align__(1024) uint8_t beam_smem[];
    uint64_t *full = reinterpret_cast<uint64_t *>(beam_smem + beam_attn_smem<T, HD, RWP, RWS>() - kBaTail);
    uint64_t *empty = full + S;
    float2 *bml = reinterpret_cast<float2 *>(empty + S);
    const uint32_t smem = smem_u32(beam_smem), rows = smem + 2 * Tl::kBytes * S;
    float *buf = reinterpret_cast<float *>(beam_smem + 2 * Tl::kBytes * S);
    pdl_launch();
    if (threadIdx.x == 0) {
#pragma unroll
        for (int i = 0; i < S; ++i) {
            mbar_init(&full[i], 32);
            mbar_init(&empty[i], kBaThreads / 32);
        }
        fence_mbar_init();
    }
    BeamCursor c;
    const bool any = beam_first(a, p, c);
    __syncthreads();
    if (!any) return;
    uint32_t s = 0, phase = 0;
    if (threadIdx.x >= kBaThreads) {
        uint32_t issued = 0;
        bool ok = true;
        // stages that 16-byte copies have filled are the copy engine's next
        const bool mixed = p.tma && (p.tma != 3 || a.slots);
        while (c.left) {
            if (issued >= S && !(ok = mbar_wait_warp(&empty[s], phase ^ 1, &g_beam_err, ERR_WAIT_EMPTY))) break;
            if (mixed) asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
            const uint32_t n = beam_take<T, HD>(c);
            beam_load<T, HD>(a, p, maps, c, n, smem + s * 2 * Tl::kBytes, &full[s]);
            ++issued;
            beam_advance(c, n);
            if (c.left && c.pos >= c.len) beam_next_item(a, p, c);
            if (++s == S) {
                s = 0;
                phase ^= 1;
            }
        }
        // no copy is in flight when this CTA's shared memory is given back
        for (uint32_t i = 0; i < min(issued, (uint32_t)S); ++i) {
            const uint32_t t = issued - 1 - i;
            mbar_wait(&full[t % S], t / S & 1, &g_beam_err, ERR_WAIT_DRAIN);
        }
        return;
    }
    BeamRows<T, HD> w;
    bool fresh = true, ok = true;
    uint32_t most = 0, wild = 0;
#pragma unroll 1
    while (c.left) {
        const uint32_t stage = smem + s * 2 * Tl::kBytes;
        if (RWP == RWS || c.part < a.n_group)
            beam_step<T, HD, RWP>(a, p, c, fresh, most, wild, w, stage, &full[s], &empty[s], phase, ok, rows, buf, bml);
        else
            beam_step<T, HD, RWS>(a, p, c, fresh, most, wild, w, stage, &full[s], &empty[s], phase, ok, rows, buf, bml);
        if (++s == S) {
            s = 0;
            phase ^= 1;
        }
    }
}

// A row by plain fp32 arithmetic, V dimensions a lane; warp w of WPR takes
// every WPR-th four positions, whose loads overlap.  For rows that the kernels'
// arithmetic cannot form, which the joining kernel finds by its partial results:
// - fp32: an infinite operand, or one within 2^-12 of the largest float, has no
//   split into two tf32 numbers (infinity minus infinity); the products are NaN.
// - scores of 2^16 and more in units of log2, keys near the largest float among
//   them: a maximum is a scaled score as rounded, and the exact product that a
//   fused multiply-add takes differs from it by up to 2^-24 of it.  That shifts
//   a row's probabilities by a common factor, which for still larger scores is
//   a power of two past the types' range.  (Rounding every product in the
//   kernels: 64 bf16 samples 147 us for 134.)
// Rare and slow: 4 fp32 beams over 8000 positions 465 us for 28.  A row that a
// NaN score has spoilt for good ends early.
template <typename T, int V, int WPR>
__device__ __forceinline__ void beam_row_plain(const BeamAttnArgs &a, uint32_t s, uint32_t t, uint32_t h, uint32_t kvh,
                                               uint32_t w, float &m, float &l, float *o) {
    const uint32_t grp = s / a.n_beam, d0 = (threadIdx.x & 31) * V;
    const bool held = d0 < a.hd;
    struct alignas(sizeof(T) * V) Vec { T v[V]; };
    auto row = [&](const void *base, size_t at, float *x) {
        Vec r{};
        if (held) r = *reinterpret_cast<const Vec *>(static_cast<const T *>(base) + at + d0);
#pragma unroll
        for (int i = 0; i < V; ++i) x[i] = beam_to_f32(r.v[i]);
    };
    float q[V];
    row(a.q, s * a.q_seq + t * a.q_tok + h * a.q_head, q);
#pragma unroll
    for (int i = 0; i < V; ++i) {
        q[i] *= a.scale;
        o[i] = 0.f;
    }
    m = -INFINITY;
    l = 0.f;
    const uint32_t np = beam_part_len(a, grp), ns = beam_part_len(a, a.n_group + s), hidden = a.n_query - 1 - t;
    const uint32_t n = np + (ns > hidden ? ns - hidden : 0);
#pragma unroll 1
    for (uint32_t j0 = 4 * w; j0 < n && l == l; j0 += 4 * WPR) {
        float k[4][V], v[4][V], x[4];
#pragma unroll
        for (int u = 0; u < 4; ++u) {
            const uint32_t j = min(j0 + u, n - 1), r = j - np;
            if (j < np) {
                const size_t at = grp * a.p_group + kvh * a.p_head + j * a.p_pos;
                row(a.pk, at, k[u]);
                row(a.pv, at, v[u]);
            } else {
                uint32_t from = s;
                if (a.slots) {
                    const uint32_t b = (uint32_t)a.slots[s * a.slot_seq + r];
                    if (b < a.n_beam) from = grp * a.n_beam + b;
                }
                const size_t at = from * a.s_seq + kvh * a.s_head + r * a.s_pos;
                row(a.sk, at, k[u]);
                row(a.sv, at, v[u]);
            }
            x[u] = 0.f;
#pragma unroll
            for (int i = 0; i < V; ++i) x[u] = fmaf(q[i], k[u][i], x[u]);
        }
#pragma unroll
        for (int d = 16; d; d >>= 1)
#pragma unroll
            for (int u = 0; u < 4; ++u) x[u] += __shfl_xor_sync(0xffffffffu, x[u], d);
#pragma unroll
        for (int u = 0; u < 4; ++u) {
            if (j0 + u >= n) break;
            x[u] = __fmul_rn(x[u], 1.4426950408889634f);  // (rounded here, so that the maximum minus itself is 0)
            const float mn = fmaxf(m, x[u]), safe = mn == -INFINITY ? 0.f : mn;
            const float al = exp2_fast(m - safe), p = exp2_fast(x[u] - safe);
            m = mn;
            l = fmaf(l, al, p);
#pragma unroll
            for (int i = 0; i < V; ++i) o[i] = fmaf(o[i], al, p * v[u][i]);
        }
    }
    if (l != l)
#pragma unroll
        for (int i = 0; i < V; ++i) o[i] = l;
}

// Joins a row's partial results.  WPR warps a row (token and head) take its
// segments in turn, four at a time, lanes the dimensions; their results are
// joined through shared memory.  More where the rows are few and so have many
// segments each; a block has one row, or eight with one warp each.
template <int WPR>
constexpr int kBjThreads = WPR > 1 ? 32 * WPR : 256;
template <typename T, int HD, int WPR>
__global__ void __launch_bounds__(kBjThreads<WPR>) beam_attn_join_kernel(BeamAttnArgs a, BeamAttnPlan p) {
    constexpr int V = HD / 32, RPB = kBjThreads<WPR> / 32 / WPR;  // rows of a block
    struct alignas(4 * V) Vec { float v[V]; };
    __shared__ Vec part[WPR > 1 ? WPR : 1][32];
    __shared__ float pm[WPR], pl[WPR];
    const uint32_t lane = threadIdx.x & 31, warp = threadIdx.x >> 5, w = warp % WPR;
    const uint32_t row = blockIdx.x * RPB + warp / WPR;
    if (row >= a.n_group * a.n_beam * a.n_query * a.n_head) return;  // (one row per block where there is a barrier)
    const uint32_t st = row / a.n_head, h = row - st * a.n_head, kvh = beam_div(h, p.by_gq), hg = h - kvh * a.gq;
    const uint32_t s = st / a.n_query, t = st - s * a.n_query, grp = s / a.n_beam;
    const uint32_t pr = ((s - grp * a.n_beam) * a.n_query + t) * a.gq + hg, sr = t * a.gq + hg;
    const uint32_t ptile = pr / p.prow, stile = sr / p.srow;
    const uint32_t pi = (grp * a.n_kv + kvh) * p.ptiles + ptile, si = (s * a.n_kv + kvh) * p.stiles + stile;
    const bool some_p = beam_part_len(a, grp) != 0, some_s = beam_part_len(a, a.n_group + s) != 0;
    pdl_wait();
    uint2 pc = make_uint2(1, 0), sc = make_uint2(1, 0);
    if (some_p) pc = p.pcta[pi];
    if (some_s) sc = p.scta[si];
    // (after a wait that ran out these may be anything)
    if (pc.y >= p.ctas || pc.x > pc.y) pc = make_uint2(1, 0);
    if (sc.y >= p.ctas || sc.x > sc.y) sc = make_uint2(1, 0);
    const uint32_t np = pc.y + 1 - pc.x, n = np + (sc.y + 1 - sc.x);
    // the rows' first slots: of a prefix segment j, and of a suffix segment
    const size_t prow = (size_t)(pi + pc.x) * p.prow + (pr - ptile * p.prow);
    const size_t srow = (size_t)(si + sc.x) * p.srow + (sr - stile * p.srow);
    float m = -INFINITY, l = 0.f;
    uint32_t wild = 0;
    Vec o{};
    for (uint32_t j0 = w; j0 < n; j0 += 4 * WPR) {
        float2 ml[4];
        Vec v[4];
#pragma unroll
        for (int u = 0; u < 4; ++u) {
            const uint32_t j = min(j0 + u * WPR, n - 1);
            const size_t at = j < np ? prow + (size_t)j * p.prow : srow + (size_t)(j - np) * p.srow;
            ml[u] = (j < np ? p.pml : p.sml)[at];
            v[u] = *reinterpret_cast<const Vec *>((j < np ? p.po : p.so) + at * HD + lane * V);
        }
#pragma unroll
        for (int u = 0; u < 4; ++u) {
            if (j0 + u * WPR >= n) break;
            const float mn = fmaxf(m, ml[u].x), safe = mn == -INFINITY ? 0.f : mn;
            const float mine = exp2_fast(m - safe), other = exp2_fast(ml[u].x - safe);
            m = mn;
            l = l * mine + fabsf(ml[u].y) * other;
            wild |= __float_as_uint(ml[u].y);
#pragma unroll
            for (int i = 0; i < V; ++i) o.v[i] = o.v[i] * mine + v[u].v[i] * other;
        }
    }
    bool again = !(l < INFINITY) || (l > 0.f && fabsf(m) > 65536.f);
    if constexpr (sizeof(T) == 4)
#pragma unroll
        for (int i = 0; i < V; ++i) again |= o.v[i] != o.v[i];  // (past head_dim: zeros)
    if constexpr (WPR > 1) {
        part[w][lane] = o;
        if (lane == 0) { pm[w] = m; pl[w] = __uint_as_float(__float_as_uint(l) | (wild & 0x80000000u)); }
        if (__syncthreads_or(again)) {
            beam_row_plain<T, V, WPR>(a, s, t, h, kvh, w, m, l, o.v);
            wild = 0;
            part[w][lane] = o;
            if (lane == 0) { pm[w] = m; pl[w] = l; }
            __syncthreads();
        }
        if (w) return;
        m = -INFINITY;
#pragma unroll
        for (int u = 0; u < WPR; ++u) m = fmaxf(m, pm[u]);
        const float safe = m == -INFINITY ? 0.f : m;
        l = 0.f;
        o = Vec{};
#pragma unroll
        for (int u = 0; u < WPR; ++u) {
            const float f = exp2_fast(pm[u] - safe);
            const Vec x = part[u][lane];
            l += fabsf(pl[u]) * f;
            wild |= __float_as_uint(pl[u]);
#pragma unroll
            for (int i = 0; i < V; ++i) o.v[i] += x.v[i] * f;
        }
    } else if (__any_sync(0xffffffffu, again)) {
        beam_row_plain<T, V, 1>(a, s, t, h, kvh, 0, m, l, o.v);
        wild = 0;
    }
    if (wild >> 31) {
        // values of suffix positions that other tokens do not see were left out:
        // this token's are added, whatever their weight
        const uint32_t len = beam_part_len(a, a.n_group + s), hidden = a.n_query - 1 - t;
        for (uint32_t r = 0; r + hidden < len; ++r) {
            uint32_t from = s;
            if (a.slots) {
                const uint32_t b = (uint32_t)a.slots[s * a.slot_seq + r];
                if (b < a.n_beam) from = grp * a.n_beam + b;
            }
            const T *v = static_cast<const T *>(a.sv) + from * a.s_seq + kvh * a.s_head + r * a.s_pos + lane * V;
#pragma unroll
            for (int i = 0; i < V; ++i)
                if (lane * V + i < a.hd) {
                    const float x = beam_to_f32(v[i]);
                    if (!isfinite(x)) o.v[i] += x;
                }
        }
    }
    T *out = static_cast<T *>(a.out) + (size_t)row * a.hd;
#pragma unroll
    for (int i = 0; i < V; ++i)
        if (lane * V + i < a.hd) out[lane * V + i] = beam_from_f32<T>(l == 0.f ? 0.f : o.v[i] / l);
    if (a.lse && lane == 0) a.lse[row] = l == 0.f ? -INFINITY : (m + log2f(l)) * 0.6931471805599453f;
}

}  // namespace fwb
