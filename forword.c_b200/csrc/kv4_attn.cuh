// kv4_attn.cuh — attention over the paged cache of 4-bit keys and values.
//
//     out = sum_p exp(s_p - lse) v_p,  s_p = scale q.k_p,  lse = log sum_p exp(s_p)
//
// for every query row (token x query head of a KV head) over the positions
// that its token sees.  A key is k = d_b (code - 8) in blocks b of 32, so
//
//     s_p = scale sum_b d_kb (codes_pb . q_b),   out = sum_p (exp(s_p - m) d_vb) codes_p
//
// and the products run on the codes, which 16 bits hold exactly; the scales
// multiply the 32-wide partial scores and the probabilities in fp32, and what
// comes of the latter goes into its products in two or three parts of bf16.
//
// Bound: at head_dim 128 a position is 144 bytes for a KV head, 6 cycles of an SM
// at the memory's rate, and 26 instructions of a warp, 11 cycles at the 2.3 a cycle
// that issue: large batches wait for instructions' results and for one another's
// pipes with the 16 warps an SM that 128 registers leave (integer pipe 50 % busy,
// tensor pipe 27 %, DRAM 38 %: none is full), small ones for their loads, a launch
// of one item 7.5 us.  Instances of 16 rows spill up to 300 bytes.  Positions are the rows of the m16n8k16 products and
// query rows the columns: a group's few rows fill 8 columns, and an instruction
// multiplies 256 values of K or V as they come unpacked into registers.  (On
// tcgen05 they would pass through shared memory, which pays from 64 rows on:
// kv4_attn_tc.cuh.)
//
// Work: an item is (sequence, row tile, KV head); the items' pairs of tiles of 16
// positions stand in one line that is cut evenly over the CTAs, an item's ends
// counting as `cost` of them, and a cut near an item's end moves there.  The
// eight warps of a CTA take an item's pairs in turn, each with a ring of its own
// that it fills by 16-byte copies, and join their results in shared memory at
// the item's end.  Where an item is cut, its parts go to the workspace and the
// CTA that arrives last adds them, in the order of the positions whichever
// arrives last.
//
// Measured on a B200 (us; graphs of calls on alternating inputs; heads of 128
// dimensions): 64 bf16 sequences of up to 8191 positions, 64 heads on 8, 93 (308
// MB: 3.3 TB/s); one fp16 token, 32 heads on 8, at 8000 positions 14.5; one fp32
// token at 200 8.2; 9 bf16 sequences of 7 tokens at 4099 39; 64 fp32 sequences of
// up to 2000, 32 heads on 8, 48.  (With weights as one
// fp16 relative to the largest value scale 84, 14.0, 8.1, 35.1: where scales lie
// 2^14 and more apart, in blocks beside one another or in positions that only later
// tokens see, results were off by up to 400 times their bounds.)
#pragma once
#include "kv4_format.cuh"

namespace fwb {

constexpr int kKaWarps = 8, kKaThreads = 32 * kKaWarps;
constexpr uint32_t kKaPair = 2 * kKvTile;  // positions that a warp takes at a time
// Weights are formed as 2^8 exp2(score - reference), and a reference is raised
// when a score of its row exceeds it by 2^7: they stay below 2^15 (the tcgen05
// kernel's go into fp16).
constexpr float kKaHead = 8.f, kKaLazy = 7.f;

struct Kv4AttnArgs {
    const void *q;
    const uint8_t *cache;
    const int32_t *pages, *len, *n_new;
    void *out;
    float *lse;
    uint64_t q_seq, q_tok, q_head, pages_seq;  // strides in elements
    uint32_t type, n_seq, n_query, n_head, n_kv, gq, hd;
    uint32_t tpp_log2, n_page, max_pages;  // tiles of a page
    uint32_t rtiles;                       // row tiles
    uint32_t cost, snap, least, whole;     // of an item's ends; see ka_cut; worth a CTA; not worth cutting (pairs of tiles)
    float scale;
    float *po;        // [2 CTAs][rows][32 NB] parts of cut items
    float2 *pml;      // [2 CTAs][rows] their references and sums
    uint32_t *ticket; // [CTAs] zero between launches
    uint32_t *err, *wait_err;  // what the tables held; a bounded wait that ran out
};

__device__ __forceinline__ float ka_exp2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
__device__ __forceinline__ void ka_mma(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1, float c0, float c1,
                                       float c2, float c3) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%11,%12,%13};"
        : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1), "f"(c0), "f"(c1), "f"(c2), "f"(c3));
}
__device__ __forceinline__ void ka_mma(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    ka_mma(d, a, b0, b1, d[0], d[1], d[2], d[3]);
}
__device__ __forceinline__ void ka_mma_bf16(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
// The 8x8 halves that a warp holds as rows, as columns.
__device__ __forceinline__ uint32_t ka_transpose(uint32_t x) {
    uint32_t y;
    asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
    return y;
}
// (code - 8) * 2^-9 of nibbles (0, 4), (1, 5), (2, 6), (3, 7) as pairs of
// halves.  A nibble in the low bits of a half is the subnormal code * 2^-24 (16
// times that in bits 4..7), so it needs its mask and one fma, which is exact.
constexpr float kKaCode = 512.f;
__device__ __forceinline__ void ka_codes(uint32_t w, uint32_t (&h)[4]) {
    const __half2 up = __half2half2(__ushort_as_half(0x7800)), up16 = __half2half2(__ushort_as_half(0x6800)),
                  eight = __half2half2(__ushort_as_half(0xa400));  // 2^15, 2^11, -2^-6
#pragma unroll
    for (int i = 0; i < 2; ++i, w >>= 8) {
        const uint32_t lo = w & 0x000f000fu, hi = w & 0x00f000f0u;
        const __half2 a = __hfma2(*reinterpret_cast<const __half2 *>(&lo), up, eight),
                      b = __hfma2(*reinterpret_cast<const __half2 *>(&hi), up16, eight);
        h[2 * i] = *reinterpret_cast<const uint32_t *>(&a);
        h[2 * i + 1] = *reinterpret_cast<const uint32_t *>(&b);
    }
}

// The same as pairs of bf16, times 2^-6 (whose subnormals have 2^-133 for a unit).
constexpr float kKaValue = 64.f;
__device__ __forceinline__ void ka_codes_bf16(uint32_t w, uint32_t (&h)[4]) {
    const __nv_bfloat162 up = __bfloat162bfloat162(__ushort_as_bfloat16(0x7f00)), up16 = __bfloat162bfloat162(__ushort_as_bfloat16(0x7d00)),
                         eight = __bfloat162bfloat162(__ushort_as_bfloat16(0xbe00));  // 2^127, 2^123, -2^-3
#pragma unroll
    for (int i = 0; i < 2; ++i, w >>= 8) {
        const uint32_t lo = w & 0x000f000fu, hi = w & 0x00f000f0u;
        const __nv_bfloat162 a = __hfma2(*reinterpret_cast<const __nv_bfloat162 *>(&lo), up, eight),
                             b = __hfma2(*reinterpret_cast<const __nv_bfloat162 *>(&hi), up16, eight);
        h[2 * i] = *reinterpret_cast<const uint32_t *>(&a);
        h[2 * i + 1] = *reinterpret_cast<const uint32_t *>(&b);
    }
}
// The upper 16 bits of two floats, which are bf16 values, and what they leave of them.
__device__ __forceinline__ uint32_t ka_upper(float2 x) { return __byte_perm(__float_as_uint(x.x), __float_as_uint(x.y), 0x7632u); }
__device__ __forceinline__ float2 ka_left(float2 x) {
    const float2 up = make_float2(__uint_as_float(__float_as_uint(x.x) & 0xffff0000u), __uint_as_float(__float_as_uint(x.y) & 0xffff0000u));
    return __ffma2_rn(up, make_float2(-1.f, -1.f), x);
}
__device__ __forceinline__ uint32_t ka_pack_bf16(float2 x) {
    const __nv_bfloat162 h = __float22bfloat162_rn(x);
    return *reinterpret_cast<const uint32_t *>(&h);
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

// What a step needs to know of its item.
struct KaItem {
    uint32_t row0;        // its first row
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

// Where the line's even cuts fall within an item of `units` units: one in its
// first `head` + 1 moves to its beginning, one at `tail` or later to its end.
struct KaCut {
    uint32_t head, tail;
};
__device__ __forceinline__ KaCut ka_cut(uint32_t units, uint32_t snap) {
    const uint32_t head = min(snap, units / 2);
    return {head, max(units > snap ? units - snap : 0u, head + 1)};
}

struct KaScan {
    uint32_t sum[32], most[32], find[3];
};

// A CTA's way along the line of items, in units of UNIT positions, for row
// tiles of ROWS.  Every thread goes it by itself.
template <int ROWS, int UNIT>
struct KaLine {
    const Kv4AttnArgs &a;
    bool whole = false;  // items count alike, and go to a CTA each
    uint32_t total, chunk, entry, head, start, units;  // start, units: of the item
    // the item's sequence and row tile, what its rows see, and this CTA's part
    uint32_t seq, rt, first, last, from, to, tiles;
    int32_t len, fresh, limit;

    __device__ __forceinline__ KaLine(const Kv4AttnArgs &args) : a(args) {}
    __device__ __forceinline__ uint32_t units_of(uint32_t e) const {
        int32_t len, fresh, limit;
        ka_lengths(a, e / a.rtiles, len, fresh);
        return !ka_tiles<ROWS>(a, e % a.rtiles, len, fresh, limit) ? 0 : whole ? 1 : (uint32_t)(limit + UNIT - 1) / UNIT + a.cost;
    }
    // Called by all the CTA's threads (whole warps); false: no part of the line is its.
    __device__ __forceinline__ bool begin(KaScan &sh) {
        const uint32_t tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, warps = blockDim.x >> 5, entries = a.n_seq * a.rtiles,
                       per = (entries + blockDim.x - 1) / blockDim.x;
        uint32_t mine = 0, top = 0, have = 0;
        for (uint32_t e = tid * per; e < min(entries, (tid + 1) * per); ++e) {
            const uint32_t n = units_of(e);
            mine += n * a.n_kv;
            have += n ? a.n_kv : 0;
            top = max(top, n);
        }
        if (entries * a.n_kv <= gridDim.x) {
            top = __reduce_max_sync(0xffffffffu, top);
            if (lane == 0) sh.most[warp] = top;
            __syncthreads();
            for (uint32_t w = 0; w < warps; ++w) top = max(top, sh.most[w]);
            if (top <= a.whole + a.cost) {
                whole = true;
                mine = have;
            }
        }
        uint32_t before = mine;
#pragma unroll
        for (int d = 1; d < 32; d <<= 1) {
            const uint32_t x = __shfl_up_sync(0xffffffffu, before, d);
            if (lane >= (uint32_t)d) before += x;
        }
        if (lane == 31) sh.sum[warp] = before;
        __syncthreads();
        total = 0;
        uint32_t base = 0;
        for (uint32_t w = 0; w < warps; ++w) {
            if (w == warp) base = total;
            total += sh.sum[w];
        }
        before += base - mine;
        chunk = whole ? 1 : max((total + gridDim.x - 1) / gridDim.x, a.least);
        const uint64_t lo = (uint64_t)blockIdx.x * chunk;
        if (lo >= total) return false;
        if (mine && before <= lo && lo < before + mine) {
            uint32_t at = before, e = tid * per, n;
            while (at + (n = units_of(e) * a.n_kv) <= lo) at += n, ++e;
            sh.find[0] = e;
            sh.find[1] = at;
            sh.find[2] = ((uint32_t)lo - at) / (n / a.n_kv);
        }
        __syncthreads();
        entry = sh.find[0];
        head = sh.find[2];
        units = units_of(entry);
        start = sh.find[1] + head * units;
        return true;
    }
    // The item's CTAs are `first` to `last`; false where they lie past this one.
    // Otherwise it has units from..to of the item (last < this CTA: none).
    __device__ __forceinline__ bool item() {
        const KaCut cut = ka_cut(units, a.snap);
        first = (start + cut.head) / chunk;
        last = (start + cut.tail - 1) / chunk;
        if (first > blockIdx.x) return false;
        seq = entry / a.rtiles;
        rt = entry % a.rtiles;
        limit = 0;
        ka_lengths(a, seq, len, fresh);
        ka_tiles<ROWS>(a, rt, len, fresh, limit);
        tiles = (uint32_t)(limit + UNIT - 1) / UNIT;
        from = first == blockIdx.x ? 0 : min(blockIdx.x * chunk - start, tiles);
        to = last == blockIdx.x ? tiles : min((blockIdx.x + 1) * chunk - start, tiles);
        return true;
    }
    // To the next item; false at the end of this CTA's part.
    __device__ __forceinline__ bool next() {
        if (last > blockIdx.x) return false;
        start += units;
        if (start >= total) return false;
        if (++head == a.n_kv) {
            head = 0;
            do units = units_of(++entry);
            while (!units);
        }
        return true;
    }
};

// The result of a row: four dimensions from d on, and its log-sum-exp.
template <int ROWS, int UNIT>
__device__ __forceinline__ void ka_finish(const KaLine<ROWS, UNIT> &ln, uint32_t r, uint32_t d, float4 v, float2 ml) {
    const Kv4AttnArgs &a = ln.a;
    const uint32_t row = ln.rt * ROWS + r, t = row / a.gq;
    if (row >= a.n_query * a.gq || (int32_t)t >= ln.fresh) return;
    const uint64_t at = ((uint64_t)ln.seq * a.n_query + t) * a.n_head + ln.head * a.gq + row % a.gq;
    const float by = ml.y == 0.f ? 0.f : 1.f / ml.y;
    if (d < a.hd) kv4_store4(a.out, at * a.hd + d, a.type, make_float4(v.x * by, v.y * by, v.z * by, v.w * by));
    if (d == 0 && a.lse) a.lse[at] = ml.y == 0.f ? -INFINITY : (ml.x + log2f(ml.y)) * 0.69314718055994531f;
}
// A part's place: a CTA begins one cut item at most, and ends one.
template <int ROWS, int UNIT>
__device__ __forceinline__ uint64_t ka_slot(const KaLine<ROWS, UNIT> &ln, uint32_t cta) { return 2ull * cta + (cta == ln.first ? 1 : 0); }
// The parts of an item added, in the order of the positions, by thread `tid` of THREADS.
template <int NB, int THREADS, int ROWS, int UNIT>
__device__ __forceinline__ void ka_add_parts(const KaLine<ROWS, UNIT> &ln, uint32_t tid) {
    const Kv4AttnArgs &a = ln.a;
    const uint32_t rows = a.n_query * a.gq;
    for (uint32_t i = tid; i < ROWS * 8 * NB; i += THREADS) {
        const uint32_t r = i / (8 * NB), d = i % (8 * NB) * 4;
        if (ln.rt * ROWS + r >= rows) continue;
        float2 ml = {-INFINITY, 0.f};
        float4 v = {0.f, 0.f, 0.f, 0.f};
#pragma unroll 8
        for (uint32_t p = ln.first; p <= ln.last; ++p) {
            const float2 y = __ldcg(a.pml + ka_slot(ln, p) * ROWS + r);
            const float4 x = __ldcg(reinterpret_cast<const float4 *>(a.po + (ka_slot(ln, p) * ROWS + r) * (32 * NB) + d));
            const float top = fmaxf(ml.x, y.x), ref = top == -INFINITY ? 0.f : top;
            const float f0 = ka_exp2(ml.x - ref), f1 = ka_exp2(y.x - ref);
            ml = make_float2(top, ml.y * f0 + y.y * f1);
            v.x = v.x * f0 + x.x * f1;
            v.y = v.y * f0 + x.y * f1;
            v.z = v.z * f0 + x.z * f1;
            v.w = v.w * f0 + x.w * f1;
        }
        ka_finish(ln, r, d, v, ml);
    }
}

template <bool SPLIT, int NB, int NT>
struct KaSmem {
    static constexpr int kStages = NT == 2 ? 2 : 3;
    static constexpr uint32_t kRows = 8 * NT, kTile = kv4_tile(NB), kStage = 2 * kTile, kStride = 32 * NB + 4;
    static constexpr uint32_t kRing = kKaWarps * kStages * kStage, kJoin = kKaWarps * kRows * kStride * 4;
    // with an item's end, which uses the rings' memory: the warps' references and sums, their weights, the rows'
    static constexpr uint32_t kSums = kJoin, kWeights = kSums + kKaWarps * kRows * 8, kRowSums = kWeights + kKaWarps * kRows * 4,
                              kEnd = kRowSums + kRows * 8;
    static constexpr uint32_t kQueries = NT * NB * (SPLIT ? 2 : 1) * 32 * 16;  // after the ring
    static constexpr uint32_t kRingBytes = kRing > kEnd ? kRing : kEnd, kBytes = kRingBytes + kQueries;
};
// What a CTA holds besides.
template <uint32_t ROWS>
struct KaStatic {
    float qs[ROWS];  // of its queries
    KaScan scan;
    uint32_t last;
};

// H tiles of 16 positions.  (Keys' codes as they lie under a mask, with sums that
// begin at -8 in every place, cost the scores 1e-6: the tensor cores' sums
// truncate at their largest term.)  EDGE: some rows may not see all positions, or
// a tile is not there.  sq: the queries' B operand [n][hi, lo][b] for each lane.
template <bool SPLIT, int NB, int NT, int H, bool EDGE>
__device__ __forceinline__ void ka_step(const Kv4AttnArgs &args, const uint8_t *pair, const uint4 *sq, const KaItem &it,
                                        int32_t pos0, uint32_t there, const float (&qs)[NT][2], float (&o)[NT][NB][2][4],
                                        float (&mm)[NT][2], float (&thr)[NT][2], float (&l)[NT][2]) {
    constexpr uint32_t TB = kv4_tile(NB);
    const uint32_t lane = threadIdx.x & 31, g = lane >> 2, c = lane & 3;
    const uint32_t p0 = (g >> 1) + 4 * (g & 1), p1 = p0 + 8;  // the positions of this lane's rows of the scores
    float s[H][NT][4];
#pragma unroll
    for (int h = 0; h < H; ++h)
#pragma unroll
        for (int n = 0; n < NT; ++n) s[h][n][0] = s[h][n][1] = s[h][n][2] = s[h][n][3] = 0.f;
    {
        uint32_t w0[H][NB], w1[H][NB], d0[H][(NB + 1) / 2], d1[H][(NB + 1) / 2];
#pragma unroll
        for (int h = 0; h < H; ++h) {
            const uint8_t *tile = pair + h * TB;
            ka_words<NB>(tile + p0 * 16 * NB + c * 4 * NB, w0[h]);
            ka_words<NB>(tile + p1 * 16 * NB + c * 4 * NB, w1[h]);
            ka_halves<NB>(tile + kv4_codes(NB) + p0 * 2 * NB, d0[h]);
            ka_halves<NB>(tile + kv4_codes(NB) + p1 * 2 * NB, d1[h]);
        }
#pragma unroll
        for (int b = 0; b < NB; ++b) {
            uint32_t a0[H][4], a1[H][4];
            float k0[H], k1[H];
#pragma unroll
            for (int h = 0; h < H; ++h) {
                uint32_t x[4], y[4];
                ka_codes(w0[h][b], x);
                ka_codes(w1[h][b], y);
                a0[h][0] = x[0]; a0[h][1] = y[0]; a0[h][2] = x[1]; a0[h][3] = y[1];
                a1[h][0] = x[2]; a1[h][1] = y[2]; a1[h][2] = x[3]; a1[h][3] = y[3];
                const float2 e0 = kv4_unpack(d0[h][b / 2]), e1 = kv4_unpack(d1[h][b / 2]);
                k0[h] = b % 2 ? e0.y : e0.x;
                k1[h] = b % 2 ? e1.y : e1.x;
            }
#pragma unroll
            for (int n = 0; n < NT; ++n) {
                uint4 q, r = {};
                q = sq[((n * (SPLIT ? 2 : 1)) * NB + b) * 32 + lane];
                if constexpr (SPLIT) r = sq[((n * 2 + 1) * NB + b) * 32 + lane];
#pragma unroll
                for (int h = 0; h < H; ++h) {
                    float acc[4];
                    if constexpr (SPLIT) {
                        ka_mma(acc, a0[h], r.x, r.y, 0.f, 0.f, 0.f, 0.f);
                        ka_mma(acc, a1[h], r.z, r.w);
                        ka_mma(acc, a0[h], q.x, q.y);
                    } else {
                        ka_mma(acc, a0[h], q.x, q.y, 0.f, 0.f, 0.f, 0.f);
                    }
                    ka_mma(acc, a1[h], q.z, q.w);
                    s[h][n][0] = fmaf(k0[h], acc[0], s[h][n][0]);
                    s[h][n][1] = fmaf(k0[h], acc[1], s[h][n][1]);
                    s[h][n][2] = fmaf(k1[h], acc[2], s[h][n][2]);
                    s[h][n][3] = fmaf(k1[h], acc[3], s[h][n][3]);
                }
            }
        }
    }
    bool raise = false;
#pragma unroll
    for (int h = 0; h < H; ++h)
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                if constexpr (EDGE) {
                    const int32_t lim = ka_limit(args, it.len, it.fresh, it.row0 + n * 8 + 2 * c + (i & 1));
                    if (!(there >> h & 1) || pos0 + (int32_t)(16 * h + (i < 2 ? p0 : p1)) >= lim) s[h][n][i] = -INFINITY;
                }
                // (thr: the same in terms of the bare score, where there are registers for it)
                raise |= NT == 1 ? s[h][n][i] > thr[n][i & 1] : fmaf(s[h][n][i], qs[n][i & 1], -mm[n][i & 1]) > kKaHead + kKaLazy;
            }
    // A row's reference follows its scores only when one of them exceeds it by 2^7
    // (its own: what other rows see changes nothing).
    if (__any_sync(0xffffffffu, raise)) {
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
            for (int j = 0; j < 2; ++j) {
                float top = fmaxf(s[0][n][j], s[0][n][j + 2]);
                if constexpr (H == 2) top = fmaxf(top, fmaxf(s[H - 1][n][j], s[H - 1][n][j + 2]));
                top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 4));
                top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 8));
                top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 16));
                const float now = fmaf(top, qs[n][j], -kKaHead);
                const bool own = NT == 1 ? top > thr[n][j] : fmaf(top, qs[n][j], -mm[n][j]) > kKaHead + kKaLazy;
                if (own && now > mm[n][j]) {
                    const float f = ka_exp2(mm[n][j] - now);
                    mm[n][j] = now;
                    thr[n][j] = (now + (kKaHead + kKaLazy)) / qs[n][j];
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
    for (int h = 0; h < H; ++h)
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                float p = ka_exp2(fmaf(s[h][n][i], qs[n][i & 1], -mm[n][i & 1]));
                if constexpr (EDGE)
                    if (s[h][n][i] == -INFINITY) p = 0.f;
                s[h][n][i] = p;
                l[n][i & 1] += p;
            }
    // The values' scales; what lies past the last row's positions is anything.
    uint32_t v[H][NB][2];  // of positions (c, c + 4) and (c + 8, c + 12): the rows of the transposed weights
#pragma unroll
    for (int h = 0; h < H; ++h) {
        const uint8_t *vd = pair + h * TB + 2 * kv4_codes(NB) + kv4_scales(NB);
        uint32_t d[4][(NB + 1) / 2];
#pragma unroll
        for (int j = 0; j < 4; ++j) ka_halves<NB>(vd + (c + 4 * j) * 2 * NB, d[j]);
        uint32_t m0 = 0xffffffffu, m1 = 0xffffffffu;
        if constexpr (EDGE) {
            const int32_t left = there >> h & 1 ? it.limit - pos0 - (int32_t)(16 * h + c) : 0;
            m0 = (left > 0 ? 0xffffu : 0u) | (left > 4 ? 0xffff0000u : 0u);
            m1 = (left > 8 ? 0xffffu : 0u) | (left > 12 ? 0xffff0000u : 0u);
        }
#pragma unroll
        for (int b = 0; b < NB; ++b) {
            const uint32_t pick = b % 2 ? 0x7632u : 0x5410u;
            v[h][b][0] = __byte_perm(d[0][b / 2], d[1][b / 2], pick) & m0;
            v[h][b][1] = __byte_perm(d[2][b / 2], d[3][b / 2], pick) & m1;
        }
    }
    // A weight times its scale goes into the products as parts in bf16, whose range is
    // fp32's: neither a row's small scales nor a block's vanish beside larger ones (as
    // fp16, with a reference of the largest scale, those 2^-14 of it and less lost bits).
#pragma unroll
    for (int h = 0; h < H; ++h) {
        // the weights' transposes: rows as columns g, positions as above (moved as two halves of their 32 bits)
        float2 w[NT][2];
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                const uint32_t x = __float_as_uint(s[h][n][2 * e]), y = __float_as_uint(s[h][n][2 * e + 1]),
                               up = ka_transpose(__byte_perm(x, y, 0x7632u)), low = ka_transpose(__byte_perm(x, y, 0x5410u));
                w[n][e] = make_float2(__uint_as_float(__byte_perm(low, up, 0x5410u)), __uint_as_float(__byte_perm(low, up, 0x7632u)));
            }
        uint32_t mask[NT][2];
        if constexpr (EDGE)
#pragma unroll
            for (int n = 0; n < NT; ++n) {
                const int32_t lim = ka_limit(args, it.len, it.fresh, it.row0 + n * 8 + g);
                const int32_t left = there >> h & 1 ? lim - pos0 - (int32_t)(16 * h + c) : 0;
                mask[n][0] = (left > 0 ? 0xffffu : 0u) | (left > 4 ? 0xffff0000u : 0u);
                mask[n][1] = (left > 8 ? 0xffffu : 0u) | (left > 12 ? 0xffff0000u : 0u);
            }
        const uint8_t *vt = pair + h * TB + kv4_codes(NB) + kv4_scales(NB);
        uint32_t u[4][(NB + 1) / 2];
#pragma unroll
        for (int j = 0; j < 4; ++j) ka_halves<NB>(vt + (c + 4 * j) * 16 * NB + (g ^ (c & 2 ? 4u : 0u)) * 2 * NB, u[j]);
#pragma unroll
        for (int b = 0; b < NB; ++b) {
            const uint32_t pick = b % 2 ? 0x7632u : 0x5410u;
            uint32_t x[4], y[4];
            ka_codes_bf16(__byte_perm(u[0][b / 2], u[1][b / 2], pick), x);
            ka_codes_bf16(__byte_perm(u[2][b / 2], u[3][b / 2], pick), y);
            const uint32_t a0[4] = {x[0], x[1], y[0], y[1]}, a1[4] = {x[2], x[3], y[2], y[3]};
            const float2 v0 = kv4_unpack(v[h][b][0]), v1 = kv4_unpack(v[h][b][1]);
#pragma unroll
            for (int n = 0; n < NT; ++n) {
                const float2 f0 = __fmul2_rn(w[n][0], v0), f1 = __fmul2_rn(w[n][1], v1), r0 = ka_left(f0), r1 = ka_left(f1);
                // 8 bits and the rest: 8 and 8 bits in fp32 calls, all of it; 8 with a rounding, 2^-17, in the others
                uint32_t p[3][2] = {{ka_upper(f0), ka_upper(f1)}, {}, {}};
                if constexpr (SPLIT) {
                    p[1][0] = ka_upper(r0);
                    p[1][1] = ka_upper(r1);
                    p[2][0] = ka_pack_bf16(ka_left(r0));
                    p[2][1] = ka_pack_bf16(ka_left(r1));
                } else {
                    p[1][0] = ka_pack_bf16(r0);
                    p[1][1] = ka_pack_bf16(r1);
                }
                constexpr int kParts = SPLIT ? 3 : 2;
                if constexpr (EDGE)  // (a scale may be NaN)
#pragma unroll
                    for (int i = 0; i < kParts; ++i) {
                        p[i][0] &= mask[n][0];
                        p[i][1] &= mask[n][1];
                    }
                if constexpr (SPLIT) {
                    // sums of 16 positions added in rounded fp32: the tensor cores' own additions truncate
                    float t0[4] = {0.f, 0.f, 0.f, 0.f}, t1[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
                    for (int i = kParts - 1; i >= 0; --i) {
                        ka_mma_bf16(t0, a0, p[i][0], p[i][1]);
                        ka_mma_bf16(t1, a1, p[i][0], p[i][1]);
                    }
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        o[n][b][0][i] += t0[i];
                        o[n][b][1][i] += t1[i];
                    }
                } else {
#pragma unroll
                    for (int i = kParts - 1; i >= 0; --i) {
                        ka_mma_bf16(o[n][b][0], a0, p[i][0], p[i][1]);
                        ka_mma_bf16(o[n][b][1], a1, p[i][0], p[i][1]);
                    }
                }
            }
        }
    }
}

// SPLIT: fp32 calls, whose queries go through the products as two halves and
// whose weights as three parts.  NT: column tiles of 8 query rows.
template <bool SPLIT, int NB, int NT>
__global__ void __launch_bounds__(kKaThreads, NT <= 2 ? 2 : 1) kv4_attn_kernel(const __grid_constant__ Kv4AttnArgs a) {
    using S = KaSmem<SPLIT, NB, NT>;
    constexpr uint32_t ROWS = S::kRows;
    constexpr int kKaStages = S::kStages;
    extern __shared__ __align__(128) uint8_t ring[];
    __shared__ KaStatic<ROWS> sh;
    // two CTAs of an SM's 228 KB, 1 KB of each the system's, static memory in steps of 1 KB
    static_assert(NT > 2 || 2 * (S::kBytes + (sizeof sh + 1023) / 1024 * 1024 + 1024) <= 228 * 1024, "shared memory of two CTAs");
    float2(*const sml)[ROWS] = reinterpret_cast<float2(*)[ROWS]>(ring + S::kSums);
    float(*const sw)[ROWS] = reinterpret_cast<float(*)[ROWS]>(ring + S::kWeights);
    float2 *const srow = reinterpret_cast<float2 *>(ring + S::kRowSums);
    const uint32_t tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, c = lane & 3;
    uint4 *const sq = reinterpret_cast<uint4 *>(ring + S::kRingBytes);
    pdl_wait();

    KaLine<ROWS, kKaPair> ln(a);
    if (!ln.begin(sh.scan)) return;
    do {
        if (!ln.item()) break;
        if (ln.last >= blockIdx.x) {
            const uint32_t seq = ln.seq, rt = ln.rt, head = ln.head, from = ln.from, to = ln.to;
            const int32_t len = ln.len, fresh = ln.fresh, limit = ln.limit;
            const uint32_t rows = a.n_query * a.gq;

            // --- the warp's positions: their pages, and the first copies ---
            uint8_t *const mine_ring = ring + warp * (kKaStages * S::kStage);
            const uint32_t count = from + warp < to ? (to - from - warp + kKaWarps - 1) / kKaWarps : 0;
            const int32_t *const table = a.pages + seq * a.pages_seq;
            // where the next 32 pairs' tiles lie, in 64-byte steps from the cache's
            // beginning (each lane a pair), and which tiles of the ring's pairs there are
            constexpr uint32_t kNone = 0xffffffffu;
            uint32_t at0 = 0, at1 = 0, there = 0;
            auto fill = [&](uint32_t i) {
                if (i < count) {
                    if (i % 32 == 0) {
                        const uint32_t t = 2 * (from + warp + (i + lane) * kKaWarps);  // the first tile
                        at0 = at1 = kNone;
                        if (i + lane < count) {
                            const bool two = (t + 1) * kKvTile < (uint32_t)limit;
                            const uint32_t page0 = (uint32_t)table[t >> a.tpp_log2],
                                           page1 = two ? (uint32_t)table[(t + 1) >> a.tpp_log2] : 0,
                                           in = (1u << a.tpp_log2) - 1;
                            if (page0 < a.n_page) at0 = (((page0 * a.n_kv + head) << a.tpp_log2) + (t & in)) * (S::kTile / 64);
                            if (two && page1 < a.n_page) at1 = (((page1 * a.n_kv + head) << a.tpp_log2) + ((t + 1) & in)) * (S::kTile / 64);
                            if (page0 >= a.n_page || page1 >= a.n_page) atomicOr(a.err, kKvBadPage);
                        }
                    }
                    const uint32_t stage = i % kKaStages, s0 = __shfl_sync(0xffffffffu, at0, i % 32),
                                   s1 = __shfl_sync(0xffffffffu, at1, i % 32);
                    const bool ok0 = s0 != kNone, ok1 = s1 != kNone;
                    there = (there & ~(3u << 2 * stage)) | ((ok0 ? 1u : 0u) | (ok1 ? 2u : 0u)) << 2 * stage;
                    constexpr uint32_t kChunks = S::kTile / 16;
                    const uint8_t *src0 = a.cache + (uint64_t)s0 * 64 + lane * 16,
                                  *src1 = a.cache + (uint64_t)s1 * 64 + lane * 16 - S::kTile;
                    uint8_t *dst = mine_ring + stage * S::kStage + lane * 16;
#pragma unroll
                    for (uint32_t k = 0; k < (2 * kChunks + 31) / 32; ++k) {
                        const uint32_t c0 = k * 32 + lane;
                        if (c0 < kChunks ? ok0 : ok1 && c0 < 2 * kChunks) cp_async16(dst + k * 512, (c0 < kChunks ? src0 : src1) + k * 512);
                    }
                }
                cp_async_commit();
            };
#pragma unroll
            for (uint32_t i = 0; i < kKaStages - 1; ++i) fill(i);

            // --- queries: the products' B operand, columns of 8 rows ---
            // 16 threads a row, 8 dimensions each.  A row is taken times a power
            // of two, its largest value in [2^13, 2^14).
            for (uint32_t i = tid; i < ROWS * 16; i += kKaThreads) {
                const uint32_t r = i / 16, ch = i % 16, b = ch / 4, row = rt * ROWS + r, t = row / a.gq, d = 8 * ch;
                float4 v0 = {0.f, 0.f, 0.f, 0.f}, v1 = v0;
                if (row < rows && (int32_t)t < fresh && d < a.hd) {
                    const uint64_t at = seq * a.q_seq + t * a.q_tok + (head * a.gq + row % a.gq) * a.q_head + d;
                    v0 = kv4_load4(a.q, at, a.type);
                    v1 = kv4_load4(a.q, at + 4, a.type);
                }
                const float x[8] = {v0.x, v0.y, v0.z, v0.w, v1.x, v1.y, v1.z, v1.w};
                float top = 0.f, odd = 0.f;
#pragma unroll
                for (int k = 0; k < 8; ++k) {
                    top = fmaxf(top, fabsf(x[k]));
                    odd += x[k] * 0.f;  // NaN where something is not finite
                }
#pragma unroll
                for (int k = 1; k < 16; k <<= 1) {
                    top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, k));
                    odd += __shfl_xor_sync(0xffffffffu, odd, k);
                }
                const uint32_t ex = min(max(__float_as_uint(top) >> 23, 14u), 254u);
                const float up = __uint_as_float((267u - ex) << 23);
                uint32_t hi[4], lo[4];
#pragma unroll
                for (int k = 0; k < 4; ++k) {
                    const float y0 = x[2 * k] * up, y1 = x[2 * k + 1] * up;
                    hi[k] = kv4_pack(y0, y1);
                    const float2 f = kv4_unpack(hi[k]);
                    lo[k] = kv4_pack(y0 - f.x, y1 - f.y);
                }
                if (b < NB) {
                    const uint32_t at = ((r / 8) * (SPLIT ? 2 : 1) * NB + b) * 32 + r % 8 * 4 + ch % 4;
                    sq[at] = make_uint4(hi[0], hi[1], hi[2], hi[3]);
                    if constexpr (SPLIT) sq[at + NB * 32] = make_uint4(lo[0], lo[1], lo[2], lo[3]);
                }
                // codes stand there as multiples of 2^-9
                if (ch == 0) sh.qs[r] = (__uint_as_float((ex - 13u) << 23) + (ex < 227 ? odd : NAN)) * (a.scale * 1.4426950408889634f) * kKaCode;
            }
            float qs[NT][2], mm[NT][2], thr[NT][2], l[NT][2], o[NT][NB][2][4];
            __syncthreads();
#pragma unroll
            for (int n = 0; n < NT; ++n) {
#pragma unroll
                for (int j = 0; j < 2; ++j) {
                    qs[n][j] = sh.qs[n * 8 + 2 * c + j];
                    mm[n][j] = thr[n][j] = -INFINITY;  // nothing seen yet
                    l[n][j] = 0.f;
                }
#pragma unroll
                for (int b = 0; b < NB; ++b)
#pragma unroll
                    for (int i = 0; i < 4; ++i) o[n][b][0][i] = o[n][b][1][i] = 0.f;
            }
            const KaItem it = {rt * ROWS, limit, len, fresh};
            const int32_t least = ka_limit(a, len, fresh, rt * ROWS);  // of the first row: the fewest positions

            for (uint32_t i = 0; i < count; ++i) {
                asm volatile("cp.async.wait_group %0;" ::"n"(kKaStages - 2) : "memory");
                __syncwarp();
                const uint32_t stage = i % kKaStages, ok = there >> 2 * stage & 3;
                const uint8_t *pair = mine_ring + stage * S::kStage;
                const int32_t pos0 = (int32_t)((from + warp + i * kKaWarps) * kKaPair);
                const bool edge = pos0 + (int32_t)kKaPair > least || ok != 3;
                if constexpr (NT == 1) {  // both tiles at once: one look at the references for two
                    if (edge) ka_step<SPLIT, NB, NT, 2, true>(a, pair, sq, it, pos0, ok, qs, o, mm, thr, l);
                    else ka_step<SPLIT, NB, NT, 2, false>(a, pair, sq, it, pos0, ok, qs, o, mm, thr, l);
                } else {                  // one after the other: registers
#pragma unroll 1
                    for (int h = 0; h < 2; ++h) {
                        if (edge) ka_step<SPLIT, NB, NT, 1, true>(a, pair + h * S::kTile, sq, it, pos0 + 16 * h, ok >> h, qs, o, mm, thr, l);
                        else ka_step<SPLIT, NB, NT, 1, false>(a, pair + h * S::kTile, sq, it, pos0 + 16 * h, ok >> h, qs, o, mm, thr, l);
                    }
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
                    if (g == 0) sml[warp][row] = make_float2(mm[n][j], sum);
#pragma unroll
                    for (int b = 0; b < NB; ++b)
                        *reinterpret_cast<float4 *>(so + (warp * ROWS + row) * S::kStride + 32 * b + 4 * g) =
                            make_float4(o[n][b][0][j], o[n][b][0][j + 2], o[n][b][1][j], o[n][b][1][j + 2]);
                }
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
                    sw[w][tid] = f * kKaValue;
                }
                srow[tid] = make_float2(top, sum);
            }
            __syncthreads();
            const uint32_t parts = ln.last - ln.first + 1;
            const uint64_t slot = ka_slot(ln, blockIdx.x);
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
                    ka_finish(ln, r, d, v, srow[r]);
                } else {
                    *reinterpret_cast<float4 *>(a.po + (slot * ROWS + r) * (32 * NB) + d) = v;
                    if (d == 0) a.pml[slot * ROWS + r] = srow[r];
                }
            }
            if (parts > 1) {
                __threadfence();
                __syncthreads();
                if (tid == 0) sh.last = atomicAdd(a.ticket + ln.first, 1u) == parts - 1;
                __syncthreads();
                if (sh.last) {
                    __threadfence();
                    if (tid == 0) a.ticket[ln.first] = 0;
                    ka_add_parts<NB, kKaThreads>(ln, tid);
                }
            }
            __syncthreads();  // the results are read: the rings may be filled again
        }
    } while (ln.next());
}

}  // namespace fwb
