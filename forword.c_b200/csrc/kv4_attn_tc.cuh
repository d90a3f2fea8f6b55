// kv4_attn_tc.cuh — attention of many query rows over the paged 4-bit cache on
// the 5th-generation tensor cores, for fp16 and bf16 and head_dims that fill 64
// or 128 dimensions: chunks of prompts, where kv4_attn.cuh's kernel would unpack
// every tile once for 32 rows.
//
// A CTA has 128 query rows as the M dimension of S = Q K^T (64 positions) and
// O += P V; S, O, Q and P are in tensor memory (with Q and P in shared memory a
// tile of 16 products of 64 columns took 1.1 us, most of it reading Q).  Eight
// warps unpack a tile's keys and values into shared memory (a thread a position
// and a quarter of its dimensions), four do the softmax (a thread a row), and a
// thread each issues the products of the one and the other kind (one for both
// took 1.9 us a tile for that alone).  Keys and values have rings of two tiles
// each: a tile's keys are done with as soon as its scores are formed, and the
// scores of tile i + 1 are formed while tile i's softmax runs.
//
// The scales of a position's key are taken times a power of two, which leaves the
// largest in [2^14, 2^15) and multiplies its scores in fp32: unpacked keys do not
// overflow, and lose 2^-33 of the largest at most.  A key d * (code - 8) has up to
// 15 bits and goes in as two halves, the second exactly the first's rounding (the
// first alone took 220 us for bf16's 233 below and cost scores 2^-11 of sum |q||k|,
// which a call of fewer rows, in kv4_attn.cuh, does not lose).  A position's values go in
// as they are, in two parts of bf16 that hold them exactly, and the weights in two
// parts, 16 bits of them (three of the four products are formed): with bf16's
// range neither a block's small scales nor a row's vanish beside larger ones.
// (One part of fp16 each, weights relative to the largest scale so far of all
// rows' positions: 234 us for the 245 below, and values that only later tokens
// see, or of other blocks, took bits of a result.)
//
// Bound: the chain of a tile's products, softmax and products beside its
// unpacking, 1.9 us a tile; the tensor pipe is 37 % busy, and 2.1
// instructions issue a cycle.  All roles have the softmax's 128 registers, of which
// it spills 220 bytes.  Measured on a B200: 512 tokens of 32
// fp16 heads on 8 of 128 at 8191 positions 245 us (272 TFLOP/s of the formula's,
// two and a half times that in products), bf16 233 us.
//
// The reference of a row is raised, and its part of O rescaled in tensor memory,
// only when a score of it exceeds it by 2^7 (see kv4_attn.cuh).  Values that are not
// finite would reach every row of a product, seen or not: they go in as zeros,
// and rows that see their position get NaN in their block at the end.
#pragma once
#include "kv4_attn.cuh"
#include "tcgen05.cuh"

namespace fwb {

constexpr int kKtRows = 128, kKtKeys = 64;
constexpr int kKtSoft = kKtRows, kKtMake = 4 * kKtKeys, kKtThreads = kKtSoft + kKtMake + 64;

template <int NB>
struct KtSmem {
    static constexpr int kDims = 32 * NB, kSub = kDims / 64;
    static constexpr uint32_t kSubBytes = kKtKeys * 128;               // 64 dimensions of a tile's keys or values
    static constexpr uint32_t kPart = kSub * kSubBytes;                // one half, or part, of them all
    static constexpr uint32_t kStage = 2 * kPart;                      // of keys or values
    static constexpr uint32_t kOffV = 2 * kStage, kOffTail = 4 * kStage;
};
struct KtTail {
    uint64_t kfull[2], vfull[2], sfull[2], sfree[2], pfull[2], pdone[2], qfull, ofree;
    uint32_t tmem, slast;
    alignas(16) float ek[2][kKtKeys];                  // what keys' scores are multiplied with
    alignas(8) uint8_t absent[2][8];                   // positions that are not there, a bit each
    alignas(8) uint8_t odd[2][4][8];                   // values that are not finite, by block
    KaScan scan;
};
template <int NB>
constexpr uint32_t kt_smem() { return KtSmem<NB>::kOffTail + sizeof(KtTail); }

// What a thread of the making warps reads of a position: 16 bytes of codes
// (8 for 64 dimensions) and all scales of its key and value.
template <int NB>
struct KtRaw {
    uint32_t k[NB], v[NB], dk[NB / 2], dv[NB / 2];
    bool there;
};
template <int NB>
__device__ __forceinline__ void kt_read(const uint8_t *p, uint32_t (&w)[NB]) {
    if constexpr (NB == 4) {
        const uint4 x = __ldg(reinterpret_cast<const uint4 *>(p));
        w[0] = x.x; w[1] = x.y; w[2] = x.z; w[3] = x.w;
    } else if constexpr (NB == 2) {
        const uint2 x = __ldg(reinterpret_cast<const uint2 *>(p));
        w[0] = x.x; w[1] = x.y;
    } else {
        w[0] = __ldg(reinterpret_cast<const uint32_t *>(p));
    }
}
__device__ __forceinline__ void kt_store16(uint32_t at, const uint32_t (&w)[4]) {
    asm volatile("st.shared.v4.u32 [%0], {%1,%2,%3,%4};" ::"r"(at), "r"(w[0]), "r"(w[1]), "r"(w[2]), "r"(w[3]) : "memory");
}
// fp32 accumulator, A (128 rows, K-major) and B (n columns): fp16, K-major B, for
// the scores; bf16, MN-major B, for the average.
__device__ __forceinline__ uint32_t kt_idesc(uint32_t n, bool values) {
    return 1u << 4 | (values ? 1u << 7 | 1u << 10 | 1u << 16 : 0u) | (n >> 3) << 17 | (128u >> 4) << 24;
}
// The position, of the eight of a making warp's half tile, of lanes 4 q ..: two
// neighbours lie four rows apart, so that eight lanes' 16-byte stores to swizzled
// rows fall on all banks.
__device__ __forceinline__ uint32_t kt_position(uint32_t q) { return q >> 1 | (q & 1) << 2; }
// Those of lanes' votes as a byte, a bit a position.
__device__ __forceinline__ uint8_t kt_positions(uint32_t votes) {
    uint32_t x = 0;
    if (votes)
        for (uint32_t q = 0; q < 8; ++q) x |= (votes >> 4 * q & 1) << kt_position(q);
    return (uint8_t)x;
}

// The scales of a position's key times the power of two that leaves the largest
// (finite) one in [2^14, 2^15); returns what undoes it (and the codes' 2^-9).
template <int NB>
__device__ __forceinline__ float kt_scales(const uint32_t (&raw)[NB / 2], __half2 (&d)[NB]) {
    float x[NB], top = 0.f;
#pragma unroll
    for (int b = 0; b < NB; ++b) {
        const float2 f = kv4_unpack(raw[b / 2]);
        x[b] = b % 2 ? f.y : f.x;
        if (fabsf(x[b]) < INFINITY) top = fmaxf(top, fabsf(x[b]));
    }
    const uint32_t ex = max(__float_as_uint(top) >> 23, 103u);  // (fp16's least is 2^-24)
    const float up = __uint_as_float((268u - ex) << 23);
#pragma unroll
    for (int b = 0; b < NB; ++b) d[b] = __half2half2(__float2half_rn(x[b] * up));
    return top == 0.f ? 0.f : __uint_as_float((ex - 5u) << 23);
}
// A key's codes times a scale, in two halves, to a swizzled row.
__device__ __forceinline__ void kt_key(uint32_t word, __half2 d, uint32_t at, uint32_t part) {
    uint32_t code[4], hi[4], lo[4];
    ka_codes(word, code);
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        const __half2 x = *reinterpret_cast<const __half2 *>(&code[j]), h = __hmul2(x, d), r = __hfma2(x, d, __hneg2(h));
        hi[j] = *reinterpret_cast<const uint32_t *>(&h);
        lo[j] = *reinterpret_cast<const uint32_t *>(&r);
    }
    kt_store16(at, hi);
    kt_store16(at + part, lo);
}
// A value's in two parts of bf16.  The scale has 11 bits: 8 and what is left; the
// first product rounded to 8, and what is left of both, which 8 hold: exact.
__device__ __forceinline__ void kt_value(uint32_t word, float scale, uint32_t at, uint32_t part) {
    const __nv_bfloat16 up = __float2bfloat16_rn(scale);
    const __nv_bfloat162 d = __bfloat162bfloat162(up), e = __float2bfloat162_rn(scale - __bfloat162float(up));
    uint32_t code[4], hi[4], lo[4];
    ka_codes_bf16(word, code);
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        const __nv_bfloat162 x = *reinterpret_cast<const __nv_bfloat162 *>(&code[j]), h = __hmul2(x, d),
                             r = __hfma2(x, e, __hfma2(x, d, __hneg2(h)));
        hi[j] = *reinterpret_cast<const uint32_t *>(&h);
        lo[j] = *reinterpret_cast<const uint32_t *>(&r);
    }
    kt_store16(at, hi);
    kt_store16(at + part, lo);
}
// A position's quarter of keys into a stage; eight positions a warp at a time.
template <int NB>
__device__ __forceinline__ float kt_make_keys(const KtRaw<NB> &raw, uint32_t stage, uint32_t p, uint32_t c) {
    using S = KtSmem<NB>;
    __half2 d[NB];
    const float ek = kt_scales<NB>(raw.dk, d);
#pragma unroll
    for (int b = 0; b < NB; ++b)
        kt_key(raw.k[b], d[b], stage + p * 128 + (b / 2) * S::kSubBytes + (((4 * (b % 2) + c) ^ (p & 7)) << 4), S::kPart);
    return ek;
}
// Its values, and what the softmax needs of the position (which stays until the
// tile's weights are used, as its values do; its keys go earlier).
template <int NB>
__device__ __forceinline__ void kt_make_values(const KtRaw<NB> &raw, float ek, uint32_t stage, KtTail &t, uint32_t s, uint32_t p, uint32_t c) {
    using S = KtSmem<NB>;
    uint32_t odd = 0;
    const uint32_t chunk = c ^ (p & 2);  // units 2c and 2c + 1 as they lie: dimensions 8 chunk.. of every block
#pragma unroll
    for (int b = 0; b < NB; ++b) {       // (of the eight: (0, 4), (1, 5), (2, 6), (3, 7))
        const float2 f = kv4_unpack(raw.dv[b / 2]);
        float d = (b % 2 ? f.y : f.x) * kKaValue;
        if (!(fabsf(d) < INFINITY)) {
            odd |= 1u << b;
            d = 0.f;
        }
        kt_value(__byte_perm(raw.v[b / 2], raw.v[NB / 2 + b / 2], b % 2 ? 0x7632u : 0x5410u), d,
                 stage + p * 128 + (b / 2) * S::kSubBytes + (((4 * (b % 2) + chunk) ^ (p & 7)) << 4), S::kPart);
    }
    if (c == 0) t.ek[s][p] = ek;
    const uint32_t gone = __ballot_sync(0xffffffffu, !raw.there), any = __ballot_sync(0xffffffffu, odd != 0);
    uint32_t bad[4] = {0, 0, 0, 0};
    if (any)
#pragma unroll
        for (int b = 0; b < NB; ++b) bad[b] = __ballot_sync(0xffffffffu, odd >> b & 1);
    if (threadIdx.x % 32 == 0) {
        t.absent[s][p / 8] = kt_positions(gone);
#pragma unroll
        for (int b = 0; b < 4; ++b) t.odd[s][b][p / 8] = kt_positions(bad[b]);
    }
}

template <typename T, int NB>
__global__ void __launch_bounds__(kKtThreads, 1) kv4_attn_tc_kernel(const __grid_constant__ Kv4AttnArgs a) {
    using S = KtSmem<NB>;
    constexpr uint32_t kTmem = 512, kO = 2 * kKtKeys, kQ = kO + 128, kP = kQ + 64;  // columns: scores, O, queries, weights (128)
    extern __shared__ __align__(1024) uint8_t kt_sm[];
    KtTail &t = *reinterpret_cast<KtTail *>(kt_sm + S::kOffTail);
    const uint32_t tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    pdl_wait();
    KaLine<kKtRows, kKtKeys> ln(a);
    if (!ln.begin(t.scan)) return;
    if (tid == 0) {
        for (int i = 0; i < 2; ++i) {
            mbar_init(&t.kfull[i], kKtMake / 32);
            mbar_init(&t.vfull[i], kKtMake / 32);
            mbar_init(&t.sfull[i], 1);
            mbar_init(&t.sfree[i], kKtSoft / 32);
            mbar_init(&t.pfull[i], kKtSoft / 32);
            mbar_init(&t.pdone[i], 1);
        }
        mbar_init(&t.qfull, kKtSoft / 32);
        mbar_init(&t.ofree, kKtSoft / 32);
        fence_mbar_init();
    }
    if (warp == (kKtSoft + kKtMake) / 32) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&t.tmem)), "r"(kTmem) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    bt_fence_before();
    __syncthreads();
    bt_fence_after();
    const uint32_t tmem = t.tmem, smem = smem_u32(kt_sm);
    bool ok = true;
    uint32_t i = 0, seg = 0;  // tiles, and items that have any, so far

    if (warp >= kKtSoft / 32 && warp < (kKtSoft + kKtMake) / 32) {
        // --- making: keys and values of a tile ---
        const uint32_t c = tid & 3, page_log2 = a.tpp_log2 + 4, p = (warp - kKtSoft / 32) * 8 + kt_position(lane >> 2);
        do {
            if (!ln.item()) break;
            if (ln.last < blockIdx.x) continue;
            const int32_t *const table = a.pages + ln.seq * a.pages_seq;
            auto page_of = [&](uint32_t tile) -> uint32_t {
                const uint32_t pos = tile * kKtKeys + p;
                return tile < ln.to && pos < (uint32_t)ln.limit ? (uint32_t)table[pos >> page_log2] : 0xffffffffu;
            };
            auto read = [&](uint32_t tile, uint32_t page) {
                KtRaw<NB> r;
                const uint32_t pos = tile * kKtKeys + p, in = pos & ((1u << page_log2) - 1), q = pos % kKvTile;
                r.there = page < a.n_page;
#pragma unroll
                for (int b = 0; b < NB; ++b) r.k[b] = r.v[b] = 0;
#pragma unroll
                for (int b = 0; b < NB / 2; ++b) r.dk[b] = r.dv[b] = 0;
                if (r.there) {
                    const uint8_t *at = a.cache + ((((uint64_t)page * a.n_kv + ln.head) << a.tpp_log2) + in / kKvTile) * kv4_tile(NB);
                    kt_read<NB>(at + q * 16 * NB + c * 4 * NB, r.k);
                    kt_read<NB / 2>(at + kv4_codes(NB) + q * 2 * NB, r.dk);
                    at += kv4_codes(NB) + kv4_scales(NB);
                    kt_read<NB>(at + q * 16 * NB + c * 4 * NB, r.v);
                    kt_read<NB / 2>(at + kv4_codes(NB) + q * 2 * NB, r.dv);
                } else if (tile < ln.to && pos < (uint32_t)ln.limit && c == 0) {
                    atomicOr(a.err, kKvBadPage);
                }
                return r;
            };
            KtRaw<NB> next = read(ln.from, page_of(ln.from));
            uint32_t page = page_of(ln.from + 1);
            for (uint32_t tile = ln.from; tile < ln.to; ++tile, ++i) {
                const uint32_t s = i & 1;
                const KtRaw<NB> now = next;
                if (tile + 1 < ln.to) {
                    next = read(tile + 1, page);
                    page = page_of(tile + 2);
                }
                // keys once the scores of the tile before last are formed, values once its weights are used
                if (i >= 2) ok = mbar_wait_warp(&t.sfull[s], (i >> 1 & 1) ^ 1, a.wait_err, ERR_WAIT_EMPTY) && ok;
                const float ek = kt_make_keys<NB>(now, smem + s * S::kStage, p, c);
                bt_fence_proxy();
                __syncwarp();
                if (lane == 0) mbar_arrive(&t.kfull[s]);
                if (i >= 2) ok = mbar_wait_warp(&t.pdone[s], (i >> 1 & 1) ^ 1, a.wait_err, ERR_WAIT_EMPTY) && ok;
                kt_make_values<NB>(now, ek, smem + S::kOffV + s * S::kStage, t, s, p, c);
                bt_fence_proxy();
                __syncwarp();
                if (lane == 0) mbar_arrive(&t.vfull[s]);
            }
        } while (ln.next());
    } else if (warp == (kKtSoft + kKtMake) / 32) {
        // --- S = Q K^T ---
        if (lane == 0) {
            const uint32_t ids = kt_idesc(kKtKeys, false);
            do {
                if (!ln.item()) break;
                if (ln.last < blockIdx.x || ln.from >= ln.to) continue;
                const uint32_t end = i + (ln.to - ln.from);
                ok = mbar_wait(&t.qfull, seg & 1, a.wait_err, ERR_WAIT_FULL) && ok;
                ++seg;
                for (; i < end; ++i) {
                    const uint32_t b = i & 1, ph = i >> 1 & 1, k = smem + b * S::kStage;
                    ok = mbar_wait(&t.kfull[b], ph, a.wait_err, ERR_WAIT_FULL) && ok;
                    if (i >= 2) ok = mbar_wait(&t.sfree[b], ph ^ 1, a.wait_err, ERR_WAIT_EMPTY) && ok;
                    bt_fence_after();
                    bt_fence_proxy();
                    if (ok)
#pragma unroll
                        for (int h = 1; h >= 0; --h)
#pragma unroll
                            for (int d = 0; d < S::kDims / 16; ++d)
                                bt_mma_ta(tmem + b * kKtKeys, tmem + kQ + d * 8,
                                          bt_desc(k + h * S::kPart + (d / 4) * S::kSubBytes + (d % 4) * 32, 16), ids,
                                          d != 0 || h != 1);
                    bt_commit(&t.sfull[b]);
                }
            } while (ln.next());
        }
        __syncwarp();
    } else if (warp == (kKtSoft + kKtMake) / 32 + 1) {
        // --- O += P V ---
        if (lane == 0) {
            const uint32_t ido = kt_idesc(S::kDims, true);
            do {
                if (!ln.item()) break;
                if (ln.last < blockIdx.x || ln.from >= ln.to) continue;
                const uint32_t n = ln.to - ln.from;
                if (seg) ok = mbar_wait(&t.ofree, (seg - 1) & 1, a.wait_err, ERR_WAIT_EMPTY) && ok;
                ++seg;
                for (uint32_t k = 0; k < n; ++k, ++i) {
                    const uint32_t b = i & 1, ph = i >> 1 & 1, v = smem + S::kOffV + b * S::kStage, ps = tmem + kP + b * kKtKeys;
                    ok = mbar_wait(&t.vfull[b], ph, a.wait_err, ERR_WAIT_FULL) && ok;
                    ok = mbar_wait(&t.pfull[b], ph, a.wait_err, ERR_WAIT_FULL) && ok;
                    bt_fence_after();
                    bt_fence_proxy();
                    if (ok)
#pragma unroll
                        for (int h = 2; h >= 0; --h)  // the weights' and the values' second parts, then the first of both
#pragma unroll
                            for (int u = 0; u < kKtKeys / 16; ++u)
                                bt_mma_ta(tmem + kO, ps + (h == 2 ? kKtKeys / 2 : 0) + u * 8,
                                          bt_desc(v + (h == 1 ? S::kPart : 0) + u * 2048, NB == 2 ? 0 : S::kSubBytes), ido, k || u != 0 || h != 2);
                    bt_commit(&t.pdone[b]);
                }
            } while (ln.next());
        }
        __syncwarp();
    } else {
        // --- softmax: a thread a row ---
        const uint32_t r = tid, lanes = (warp * 32) << 16, mine = tmem + kO + lanes;  // mine: this row's part of O
        do {
            if (!ln.item()) break;
            if (ln.last < blockIdx.x) continue;
            const uint32_t n = ln.to - ln.from, row = ln.rt * kKtRows + r, tok = row / a.gq;
            const int32_t lim = row < a.n_query * a.gq ? ka_limit(a, ln.len, ln.fresh, row) : -1,
                          least = ka_limit(a, ln.len, ln.fresh, ln.rt * kKtRows);  // of the first row: the fewest positions
            float qs;
            {
                // the row times a power of two, its largest value in [2^13, 2^14)
                uint4 raw[S::kDims / 8];
                float top = 0.f, odd = 0.f;
                const uint64_t at = ln.seq * a.q_seq + tok * a.q_tok + (ln.head * a.gq + row % a.gq) * a.q_head;
#pragma unroll
                for (int j = 0; j < S::kDims / 8; ++j) {
                    raw[j] = make_uint4(0, 0, 0, 0);
                    if (lim >= 0 && 8 * j < a.hd) raw[j] = __ldg(reinterpret_cast<const uint4 *>(static_cast<const T *>(a.q) + at + 8 * j));
                }
#pragma unroll
                for (int j = 0; j < S::kDims / 8; ++j) {
                    float x[8];
                    kv4_floats8<T>(raw[j], x);
#pragma unroll
                    for (int e = 0; e < 8; ++e) {
                        top = fmaxf(top, fabsf(x[e]));
                        odd += x[e] * 0.f;  // NaN where something is not finite
                    }
                }
                const uint32_t ex = min(max(__float_as_uint(top) >> 23, 14u), 254u);
                const float up = __uint_as_float((267u - ex) << 23);
                qs = (__uint_as_float((ex - 13u) << 23) + (ex < 227 ? odd : NAN)) * (a.scale * 1.4426950408889634f);
#pragma unroll
                for (int j = 0; j < S::kDims / 8; j += 2) {
                    uint32_t w[8];
#pragma unroll
                    for (int h = 0; h < 2; ++h) {
                        float x[8];
                        kv4_floats8<T>(raw[j + h], x);
#pragma unroll
                        for (int e = 0; e < 4; ++e) w[4 * h + e] = kv4_pack(x[2 * e] * up, x[2 * e + 1] * up);
                    }
                    bt_st8(tmem + kQ + lanes + 4 * j, w);
                }
                bt_st_wait();
            }
            if (n) {
                bt_fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive(&t.qfull);
            }
            float ref = -INFINITY, l = 0.f;  // ref: 8 less than the row's reference
            uint32_t nan = 0;
            for (uint32_t k = 0; k < n; ++k, ++i) {
                const uint32_t b = i & 1, ph = i >> 1 & 1;
                const int32_t pos0 = (int32_t)((ln.from + k) * kKtKeys);
                ok = mbar_wait_warp(&t.sfull[b], ph, a.wait_err, ERR_WAIT_FULL) && ok;
                bt_fence_after();
                float y[kKtKeys];
                bt_ld32(tmem + b * kKtKeys + lanes, y);
                bt_ld32(tmem + b * kKtKeys + lanes + 32, y + 32);
                bt_ld_wait();
                bt_here<kKtKeys>(y);
                bt_fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive(&t.sfree[b]);
                ok = mbar_wait_warp(&t.vfull[b], ph, a.wait_err, ERR_WAIT_FULL) && ok;
                if (i >= 2) ok = mbar_wait_warp(&t.pdone[b], ph ^ 1, a.wait_err, ERR_WAIT_EMPTY) && ok;  // the weights' place is free
#pragma unroll
                for (int j = 0; j < kKtKeys; j += 4) {
                    const float4 e = *reinterpret_cast<const float4 *>(&t.ek[b][j]);
                    y[j] *= e.x; y[j + 1] *= e.y; y[j + 2] *= e.z; y[j + 3] *= e.w;
                }
                const unsigned long long absent = *reinterpret_cast<const unsigned long long *>(t.absent[b]);
                unsigned long long odds = 0;
#pragma unroll
                for (int e = 0; e < NB; ++e) odds |= *reinterpret_cast<const unsigned long long *>(t.odd[b][e]);
                const bool edge = pos0 + kKtKeys > least || absent || odds;
                if (edge) {
                    const int32_t left = lim - pos0;
                    const unsigned long long see = (left >= kKtKeys ? ~0ull : left <= 0 ? 0ull : (1ull << left) - 1) & ~absent;
                    const uint32_t see0 = (uint32_t)see, see1 = (uint32_t)(see >> 32);
#pragma unroll
                    for (int j = 0; j < kKtKeys; ++j)
                        if (!((j < 32 ? see0 : see1) >> (j % 32) & 1)) y[j] = -INFINITY;
                    if (odds)
#pragma unroll
                        for (int e = 0; e < NB; ++e)
                            if (*reinterpret_cast<const unsigned long long *>(t.odd[b][e]) & see) nan |= 1u << e;
                }
                float top = y[0];
#pragma unroll
                for (int j = 1; j < kKtKeys; ++j) top = fmaxf(top, y[j]);
                const bool own = fmaf(top, qs, -ref) > kKaHead + kKaLazy;
                if (__any_sync(0xffffffffu, own)) {
                    const float was = ref;
                    if (own) ref = fmaf(top, qs, -kKaHead);
                    const float f = own ? ka_exp2(was - ref) : 1.f;
                    l *= f;
                    if (k) {
                        ok = mbar_wait_warp(&t.pdone[b ^ 1], (i - 1) >> 1 & 1, a.wait_err, ERR_WAIT_FULL) && ok;
                        bt_fence_after();
#pragma unroll 1
                        for (uint32_t d = 0; d < S::kDims; d += 8) {
                            float o[8];
                            bt_ld8(mine + d, o);
                            bt_ld_wait();
                            bt_here<8>(o);
#pragma unroll
                            for (int e = 0; e < 8; ++e) o[e] *= f;
                            bt_st8(mine + d, o);
                        }
                        bt_st_wait();
                    }
                }
                const uint32_t ps = tmem + kP + b * kKtKeys + lanes;
#pragma unroll
                for (int j = 0; j < kKtKeys; j += 16) {
                    uint32_t w[8], r[8];
#pragma unroll
                    for (int h = 0; h < 8; ++h) {
                        float2 x;
#pragma unroll
                        for (int e = 0; e < 2; ++e) {
                            const float v = y[j + 2 * h + e];
                            float p = ka_exp2(fmaf(v, qs, -ref));
                            if (edge && v == -INFINITY) p = 0.f;
                            l += p;
                            (e ? x.y : x.x) = p;
                        }
                        w[h] = ka_upper(x);
                        r[h] = ka_pack_bf16(ka_left(x));
                    }
                    bt_st8(ps + j / 2, w);
                    bt_st8(ps + kKtKeys / 2 + j / 2, r);
                }
                bt_st_wait();
                bt_fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive(&t.pfull[b]);
            }
            // --- the item's end ---
            if (n) {
                ok = mbar_wait_warp(&t.pdone[(i - 1) & 1], (i - 1) >> 1 & 1, a.wait_err, ERR_WAIT_FULL) && ok;
                bt_fence_after();
            }
            const bool parts = ln.last > ln.first;
            const uint64_t place = ka_slot(ln, blockIdx.x) * kKtRows + r;
            const float2 ml = make_float2(ref, l);
#pragma unroll 1
            for (uint32_t d = 0; d < S::kDims; d += 8) {  // dimensions (0, 4), (1, 5), (2, 6), (3, 7) of eight
                float o[8] = {};
                if (n) {
                    bt_ld8(mine + d, o);
                    bt_ld_wait();
                    bt_here<8>(o);
                }
                float4 x = make_float4(o[0], o[2], o[4], o[6]), y = make_float4(o[1], o[3], o[5], o[7]);
                if (nan >> (d / 32) & 1) x = y = make_float4(NAN, NAN, NAN, NAN);
                if (parts) {
                    *reinterpret_cast<float4 *>(a.po + place * S::kDims + d) = x;
                    *reinterpret_cast<float4 *>(a.po + place * S::kDims + d + 4) = y;
                } else {
                    ka_finish(ln, r, d, x, ml);
                    ka_finish(ln, r, d + 4, y, ml);
                }
            }
            if (n) {
                bt_fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive(&t.ofree);
            }
            if (parts) {
                a.pml[place] = ml;
                __threadfence();
                bar_sync(1, kKtSoft);
                if (tid == 0) t.slast = atomicAdd(a.ticket + ln.first, 1u) == ln.last - ln.first;
                bar_sync(1, kKtSoft);
                if (t.slast) {
                    __threadfence();
                    if (tid == 0) a.ticket[ln.first] = 0;
                    ka_add_parts<NB, kKtSoft>(ln, tid);
                }
                bar_sync(1, kKtSoft);
            }
        } while (ln.next());
    }
    // every product is complete: the softmax waited for the last one's commit
    // (or the wait ran out after its bound)
    bt_fence_before();
    __syncthreads();
    if (warp == (kKtSoft + kKtMake) / 32) {
        bt_fence_after();
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(kTmem) : "memory");
    }
}

}  // namespace fwb
