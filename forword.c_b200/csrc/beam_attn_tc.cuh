// beam_attn_tc.cuh — the prefix part of the shared-prefix attention
// (beam_attn.cuh) on the 5th-generation tensor cores, for fp16 and bf16 and
// many rows.  The suffixes, short and with few rows each, stay with
// beam_attn.cuh's kernel, launched before this one; a CTA of each does not fit
// an SM together, so an SM takes up its prefixes when its suffixes are done.
//
// The products are transposed: a tile's 128 positions are the M dimension of
// S^T = K Q^T (N: 128 query rows), and the head's dimensions that of
// O^T += V^T P.  A thread of the softmax owns one position and half of the
// rows, so the sums over positions are kept per thread and joined once per
// item.
//
// The running maximum of a row is a reference that need not be exact: it is
// raised, and O^T rescaled in tensor memory, only when a score exceeds it by
// more than 8 in units of log2; probabilities then stay below 2^8.  So a tile
// costs no reduction over positions, only one vote of the threads that share
// the rows.
//
// Bound: per tile of 128 positions and rows the products take 1024 cycles,
// the exponentials 1024 (16 a cycle and SM), shared memory about 2000 (both
// operands of both products, the copies, P); measured 4000, with eight softmax
// warps waiting on one another and on short chains.  64 bf16 samples (512 rows
// for each of 8 KV heads) over 32763 positions: 135 us on the device with their
// suffixes, 510 TFLOP/s, against 276 with warp-level products.
//
// One CTA per SM: a warp that loads (copy engine), one thread that issues the
// products, and two groups of four warps for the softmax, each with half of
// the rows.  The scores of tile i + 1 are formed while tile i's softmax runs.
// K and V have rings of their own: a K tile is done with as soon as its
// scores are formed, so the next but one is on its way a whole softmax earlier
// than V's.
#pragma once
#include "beam_attn.cuh"

namespace fwb {

constexpr int kBtKeys = 128;
constexpr int kBtSoft = 256;                 // threads of the softmax
constexpr int kBtThreads = 64 + kBtSoft;
constexpr float kBtRaise = 8.f;              // log2
constexpr int kBtRows = 128;                 // query rows of a tile
// Minus the reference of a row that has seen no score above -inf: finite, so
// that a score of -inf stays one against it, and so large that any other
// exceeds it and raises it.
constexpr float kBtUnset = 3.4028234664e38f;

// Shared memory: two stages of K and two of V, query rows, two buffers of
// probabilities, then the small things.
template <int HD>
struct BeamTc {
    static constexpr int kSub = HD / 64;                           // sub-tiles of 128 bytes
    static constexpr uint32_t kSubBytes = kBtKeys * 128;           // of K, V
    static constexpr uint32_t kTile = kSub * kSubBytes;
    static constexpr uint32_t kQ = kBtRows * HD * 2, kP = 2 * kSubBytes;
    static constexpr uint32_t kOffV = 2 * kTile, kOffQ = 4 * kTile, kOffP = kOffQ + kQ, kOffTail = kOffP + 2 * kP;
    static constexpr uint32_t kTmem = 512;                         // a power of two, at least 3 x 128 columns
};
struct BeamTcTail {
    uint64_t kfull[2], vfull[2], kempty[2], vempty[2], sfull[2], sfree[2], pfull[2], odone[2], ofree, qfull;
    uint32_t tmem;
    alignas(16) float nm[128];  // minus the rows' references; kBtUnset: none yet
    float alpha[128];
    uint32_t top[128];          // the tile's maxima, as ordered integers; 0 between uses
};
template <int HD>
constexpr uint32_t beam_tc_smem() { return BeamTc<HD>::kOffTail + sizeof(BeamTcTail); }

// Whether a phase is over, without waiting at all.
__device__ __forceinline__ bool bt_test(uint64_t *bar, uint32_t parity) {
    uint32_t ok;
    asm volatile("{\n\t.reg .pred p;\n\tmbarrier.test_wait.parity.shared::cta.b64 p, [%1], %2;\n\tselp.u32 %0, 1, 0, p;\n\t}"
                 : "=r"(ok) : "r"(smem_u32(bar)), "r"(parity) : "memory");
    return ok != 0;
}
__device__ __forceinline__ void bt_fence_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void bt_fence_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void bt_fence_proxy() { asm volatile("fence.proxy.async.shared::cta;" ::: "memory"); }
__device__ __forceinline__ void bt_commit(uint64_t *bar) {
    asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(smem_u32(bar)) : "memory");
}
// Shared-memory matrix descriptor, 128-byte swizzle: rows of 128 bytes, eight
// of them (1024 bytes) an atom.  K-major operands: the next 8 rows 1024 bytes
// on; MN-major ones: the next 8 k 1024 bytes on, the next 64 of M or N `lead`.
__device__ __forceinline__ uint64_t bt_desc(uint32_t addr, uint32_t lead) {
    return (uint64_t)((addr & 0x3ffffu) >> 4) | (uint64_t)(lead >> 4) << 16 | (uint64_t)(1024u >> 4) << 32 |
           (uint64_t)1 << 46 | (uint64_t)2 << 61;
}
// fp32 accumulator, A and B of type T (M 128, N n), both K-major or both MN-major.
template <typename T>
__device__ __forceinline__ uint32_t bt_idesc(uint32_t n, bool mn_major) {
    const uint32_t t = beam_is_bf16(T{}) ? 1u : 0u;
    return 1u << 4 | t << 7 | t << 10 | (mn_major ? 3u << 15 : 0u) | (n >> 3) << 17 | (128u >> 4) << 24;
}
__device__ __forceinline__ void bt_mma(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, bool add) {
    asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
                 "tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}"
                 ::"r"(d), "l"(a), "l"(b), "r"(idesc), "r"((uint32_t)add) : "memory");
}

// 8 accumulator columns of this thread's lane (not waited for) / back.
__device__ __forceinline__ void bt_ld8(uint32_t addr, float *v) {
    uint32_t r[8];
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x8.b32 {%0,%1,%2,%3,%4,%5,%6,%7}, [%8];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7])
                 : "r"(addr));
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = __uint_as_float(r[i]);
}
__device__ __forceinline__ void bt_ld32(uint32_t addr, float *v) {
    uint32_t r[32];
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,"
        "%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]),
          "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]),
          "=r"(r[16]), "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]),
          "=r"(r[24]), "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
        : "r"(addr));
#pragma unroll
    for (int i = 0; i < 32; ++i) v[i] = __uint_as_float(r[i]);
}
__device__ __forceinline__ void bt_ld_wait() { asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory"); }
// Keeps uses of loaded values behind the wait before it.
template <int N>
__device__ __forceinline__ void bt_here(float *v) {
#pragma unroll
    for (int i = 0; i < N; ++i) asm volatile("" : "+f"(v[i]));
}
__device__ __forceinline__ void bt_st8(uint32_t addr, const float *v) {
    asm volatile("tcgen05.st.sync.aligned.32x32b.x8.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8};" ::"r"(addr),
                 "r"(__float_as_uint(v[0])), "r"(__float_as_uint(v[1])), "r"(__float_as_uint(v[2])),
                 "r"(__float_as_uint(v[3])), "r"(__float_as_uint(v[4])), "r"(__float_as_uint(v[5])),
                 "r"(__float_as_uint(v[6])), "r"(__float_as_uint(v[7])) : "memory");
}
__device__ __forceinline__ bool bt_any(uint32_t barrier, bool v) {  // of the 128 threads of a group
    uint32_t r;
    asm volatile("{\n\t.reg .pred p, q;\n\tsetp.ne.u32 p, %1, 0;\n\t"
                 "barrier.cta.red.or.pred q, %2, 128, p;\n\tselp.u32 %0, 1, 0, q;\n\t}"
                 : "=r"(r) : "r"((uint32_t)v), "r"(barrier) : "memory");
    return r != 0;
}

// Two fp32 at once: a = a * s + b, and a += b.
__device__ __forceinline__ void bt_fma2(float &a0, float &a1, float s, float b0, float b1) {
    asm("{\n\t.reg .b64 x, y, z;\n\tmov.b64 x, {%0, %1};\n\tmov.b64 y, {%2, %2};\n\tmov.b64 z, {%3, %4};\n\t"
        "fma.rn.f32x2 x, x, y, z;\n\tmov.b64 {%0, %1}, x;\n\t}"
        : "+f"(a0), "+f"(a1) : "f"(s), "f"(b0), "f"(b1));
}
__device__ __forceinline__ void bt_add2(float &a0, float &a1, float b0, float b1) {
    asm("{\n\t.reg .b64 x, y;\n\tmov.b64 x, {%0, %1};\n\tmov.b64 y, {%2, %3};\n\t"
        "add.rn.f32x2 x, x, y;\n\tmov.b64 {%0, %1}, x;\n\t}"
        : "+f"(a0), "+f"(a1) : "f"(b0), "f"(b1));
}

// Joins N values of every lane over the warp: each step keeps half of the
// values and hands the other half to the lane across.  Lane ends with values
// first .. first + max(1, N / 32) - 1 (lanes may hold the same ones) in v.
template <int N, int D = 16, typename Op>
__device__ __forceinline__ uint32_t bt_join(float *v, Op op) {
    uint32_t first = 0;
    if constexpr (N > 1) {
        constexpr int H = N / 2;
        const bool up = threadIdx.x & D;
#pragma unroll
        for (int j = 0; j < H; ++j) {
            const float a = v[j], b = v[j + H];
            const float give = up ? a : b, keep = up ? b : a;
            v[j] = op(keep, __shfl_xor_sync(0xffffffffu, give, D));
        }
        first = up ? H : 0;
        if constexpr (D > 1) first += bt_join<H, D / 2>(v, op);
    } else {
        v[0] = op(v[0], __shfl_xor_sync(0xffffffffu, v[0], D));
        if constexpr (D > 1) bt_join<1, D / 2>(v, op);
    }
    return first;
}

// n positions of a prefix, K or V, into a stage: by the copy engine, or where
// the strides do not allow its maps by 16-byte asynchronous copies.  The
// barrier takes 32 arrivals.
template <typename T, int HD>
__device__ __forceinline__ void bt_copy(const BeamAttnArgs &a, const BeamCursor &c, uint32_t n, bool tma, uint32_t dst,
                                        const void *base, const CUtensorMap *map, const CUtensorMap *wide, uint64_t *bar) {
    constexpr int kSub = HD / 64, CH = HD / 8, RP = 32 / CH;
    const uint32_t lane = threadIdx.x & 31, units = (n + kBaUnit - 1) / kBaUnit;
    if (tma) {
        const bool whole = units == kBtKeys / kBaUnit;  // one box per sub-tile, else one per unit and sub-tile
        if (lane == 0)
            asm volatile("mbarrier.expect_tx.relaxed.cta.shared::cta.b64 [%0], %1;" ::"r"(smem_u32(bar)),
                         "r"(units * kSub * kBaUnit * 128) : "memory");
        __syncwarp();
        const uint32_t u = lane / kSub, h = lane % kSub;
        if (u < (whole ? 1 : units))
            tma_load_4d(dst + h * (kBtKeys * 128) + u * kBaUnit * 128, whole ? wide : map, (int32_t)(h * 64),
                        (int32_t)(c.pos + u * kBaUnit), (int32_t)c.kvh, (int32_t)c.part, bar);
        mbar_arrive(bar);
        return;
    }
    const uint32_t ch = lane % CH;
    const bool held = ch * 8 < a.hd;
    const T *b = static_cast<const T *>(base) + c.part * a.p_group + c.kvh * a.p_head + (held ? ch * 8 : 0);
#pragma unroll 4
    for (uint32_t row = lane / CH; row < n; row += RP)
        cp_async16_or_zero(dst + (ch >> 3) * (kBtKeys * 128) + row * 128 + (((ch ^ row) & 7) << 4),
                           b + (size_t)(c.pos + row) * a.p_pos, held);
    asm volatile("cp.async.mbarrier.arrive.noinc.shared::cta.b64 [%0];" ::"r"(smem_u32(bar)) : "memory");
}

__device__ __forceinline__ uint32_t bt_take(const BeamCursor &c) {
    return min(min((uint32_t)kBtKeys, c.len - c.pos), min(c.left, kBtKeys / kBaUnit) * kBaUnit);
}

// The CTA's tile i by the softmax threads.
template <typename T, int HD>
__device__ __forceinline__ void bt_step(const BeamAttnArgs &a, const BeamAttnPlan &p, BeamCursor &c, bool &fresh,
                                        float *l, uint32_t i, uint8_t *sm, BeamTcTail &t, uint32_t tmem,
                                        bool &ok) {
    using Sm = BeamTc<HD>;
    constexpr int RT = kBtRows, NC = RT / 2;
    const uint32_t lane = threadIdx.x & 31, warp = threadIdx.x >> 5, quad = warp & 3, wg = (warp - 2) >> 2;
    const uint32_t tid = threadIdx.x - 64, wt = tid & 127, col0 = wg * NC, bar = 2 + wg;
    const uint32_t key = quad * 32 + lane, lanes = (quad * 32) << 16;
    const uint32_t rows = a.n_beam * a.n_query * a.gq;
    const float sl2 = a.scale * 1.4426950408889634f;
    if (fresh) {
        // query rows, K-major with the 128-byte swizzle; rows past the item's are zeros
        constexpr int CH = HD / 8, RPP = kBtSoft / CH, NR = RT / RPP;  // rows of a pass; passes
        const uint32_t qs = smem_u32(sm + Sm::kOffQ), ch = tid % CH, r0 = tid / CH;
        uint4 v[NR];
#pragma unroll
        for (int j = 0; j < NR; ++j) {
            const uint32_t r = r0 + j * RPP;
            int32_t lim;
            const T *q = beam_q_row<T, HD>(a, p, c, c.tile * RT + r, lim);
            v[j] = make_uint4(0, 0, 0, 0);  // (rows past the item's: zeros, and not written at the end)
            if (q && ch * 8 < a.hd) v[j] = *reinterpret_cast<const uint4 *>(q + ch * 8);
        }
#pragma unroll
        for (int j = 0; j < NR; ++j) {
            const uint32_t r = r0 + j * RPP;
            asm volatile("st.shared.v4.u32 [%0], {%1,%2,%3,%4};" ::"r"(qs + (ch >> 3) * (RT * 128) + r * 128 + (((ch ^ r) & 7) << 4)),
                         "r"(v[j].x), "r"(v[j].y), "r"(v[j].z), "r"(v[j].w) : "memory");
        }
        if (wt < NC) t.nm[col0 + wt] = kBtUnset;
#pragma unroll
        for (int j = 0; j < NC; ++j) l[j] = 0.f;
        bt_fence_proxy();
        bar_sync(1, kBtSoft);
        if (tid == 0) mbar_arrive(&t.qfull);
    }
    const bool first = fresh, start = c.pos == 0;
    const uint32_t n = bt_take(c), b = i & 1, ph = i >> 1 & 1;
    ok = mbar_wait_warp(&t.sfull[b], ph, &g_beam_err, ERR_WAIT_FULL) && ok;
    bt_fence_after();
    float y[NC];
    const uint32_t ts = tmem + b * RT + lanes + col0;
    const bool live = key < n;
    auto load = [&] {  // the scores
#pragma unroll
        for (int j = 0; j < NC; j += 32) bt_ld32(ts + j, y + j);
        bt_ld_wait();
        bt_here<NC>(y);
    };
    auto hide = [&] {  // positions past the end
        if (n < kBtKeys && !live)
#pragma unroll
            for (int j = 0; j < NC; ++j) y[j] = -INFINITY;
    };
    auto refer = [&] {  // against the rows' references
#pragma unroll
        for (int j = 0; j < NC; j += 4) {
            const float4 nm = *reinterpret_cast<const float4 *>(&t.nm[col0 + j]);
            bt_fma2(y[j], y[j + 1], sl2, nm.x, nm.y);
            bt_fma2(y[j + 2], y[j + 3], sl2, nm.z, nm.w);
        }
        hide();
    };
    load();
    bool raise = first;
    if (!first) {
        refer();
        float over = -INFINITY;
#pragma unroll
        for (int j = 0; j < NC; ++j) over = fmaxf(over, y[j]);
        raise = bt_any(bar, over > kBtRaise);
        if (raise) load();
    }
    if (raise) {
        hide();
        const uint32_t at = bt_join<NC>(y, [](float u, float v) { return fmaxf(u, v); });
#pragma unroll
        for (int j = 0; j < NC / 32; ++j) {
            const uint32_t u = __float_as_uint(y[j] * sl2);
            atomicMax(&t.top[col0 + at + j], u & 0x80000000u ? ~u : u | 0x80000000u);
        }
        bar_sync(bar, 128);
        if (wt < NC) {
            const uint32_t r = col0 + wt, m = t.top[r];
            t.top[r] = 0;
            const float now = fmaxf(-t.nm[r], __uint_as_float(m & 0x80000000u ? m & 0x7fffffffu : ~m));
            t.alpha[r] = exp2_fast(-t.nm[r] - now);
            t.nm[r] = -now;  // (kBtUnset while the row has seen nothing)
        }
        bar_sync(bar, 128);
        load();
        refer();
        if (!first) {  // the sums and the output so far
#pragma unroll
            for (int j = 0; j < NC; ++j) l[j] *= t.alpha[col0 + j];
            ok = mbar_wait_warp(&t.odone[(i - 1) & 1], (i - 1) >> 1 & 1, &g_beam_err, ERR_WAIT_FULL) && ok;
            bt_fence_after();
            const uint32_t to = tmem + 2 * RT + lanes + col0;
#pragma unroll 1
            for (uint32_t j = 0; j < NC; j += 8) {
                float o[8];
                bt_ld8(to + j, o);
                bt_ld_wait();
                bt_here<8>(o);
#pragma unroll
                for (int e = 0; e < 8; ++e) o[e] *= t.alpha[col0 + j + e];
                bt_st8(to + j, o);
            }
            asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory");
        }
    }
    bt_fence_before();
    __syncwarp();
    if (lane == 0) mbar_arrive(&t.sfree[b]);
    // the buffer's last reader; in order for every tile, so that the phases of
    // these barriers are never two ahead of what was seen
    if (i >= 2) ok = mbar_wait_warp(&t.odone[b], ph ^ 1, &g_beam_err, ERR_WAIT_EMPTY) && ok;
    const uint32_t ps = smem_u32(sm + Sm::kOffP + b * Sm::kP) + key * 128;
    // (in V's type, as the products take them: beam_tile has what that costs)
#pragma unroll
    for (int j = 0; j < NC; j += 8) {
        uint32_t w[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const float q0 = exp2_fast(y[j + 2 * e]), q1 = exp2_fast(y[j + 2 * e + 1]);
            bt_add2(l[j + 2 * e], l[j + 2 * e + 1], q0, q1);
            w[e] = pack2(q0, q1, T{});
        }
        const uint32_t col = col0 + j;
        asm volatile("st.shared.v4.u32 [%0], {%1,%2,%3,%4};" ::"r"(ps + (col >> 6) * Sm::kSubBytes + ((((col >> 3) ^ key) & 7) << 4)),
                     "r"(w[0]), "r"(w[1]), "r"(w[2]), "r"(w[3]) : "memory");
    }
    if (n & (kBaUnit - 1)) {
        // V rows of the last unit past the end: their probabilities are zero,
        // and zero times whatever the memory holds must be zero
        ok = mbar_wait_warp(&t.vfull[b], ph, &g_beam_err, ERR_WAIT_FULL) && ok;
        const uint32_t vs = smem_u32(sm + Sm::kOffV + b * Sm::kTile);
        const uint32_t end = (n + kBaUnit - 1) / kBaUnit * kBaUnit;
        for (uint32_t j = tid; j < (end - n) * (HD / 8); j += kBtSoft) {
            const uint32_t row = n + j / (HD / 8), ch = j % (HD / 8);
            asm volatile("st.shared.v4.u32 [%0], {%1,%1,%1,%1};" ::"r"(vs + (ch >> 3) * Sm::kSubBytes + row * 128 + ((ch & 7) << 4)),
                         "r"(0) : "memory");  // (whole rows: their swizzle does not matter)
        }
    }
    bt_fence_proxy();
    bt_fence_before();
    __syncwarp();
    if (lane == 0) mbar_arrive(&t.pfull[b]);
    beam_advance(c, n);
    fresh = c.pos >= c.len || c.left == 0;
    const uint32_t item = (c.part * a.n_kv + c.kvh) * p.ptiles + c.tile;
    if (fresh) {
        ok = mbar_wait_warp(&t.odone[b], ph, &g_beam_err, ERR_WAIT_FULL) && ok;
        bt_fence_after();
        const size_t row0 = (size_t)(item + blockIdx.x) * RT;
        float *o = p.po + row0 * HD + key;
        const uint32_t to = tmem + 2 * RT + lanes + col0, held = rows - min(rows, c.tile * RT);
#pragma unroll 1
        for (uint32_t j = 0; j < NC; j += 32) {
            float v[32];
            bt_ld32(to + j, v);
            bt_ld_wait();
            bt_here<32>(v);
            if (key < HD)
#pragma unroll
                for (int e = 0; e < 32; ++e)
                    if (col0 + j + e < held) o[(size_t)(col0 + j + e) * HD] = v[e];
        }
        bt_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&t.ofree);
        // the sums over the 128 positions, through the probabilities' place
        float *sum = reinterpret_cast<float *>(sm + Sm::kOffP);
        const uint32_t at = bt_join<NC>(l, [](float u, float v) { return u + v; });
#pragma unroll
        for (int j = 0; j < NC / 32; ++j) sum[quad * RT + col0 + at + j] = l[j];
        bar_sync(bar, 128);
        if (wt < NC && col0 + wt < held) {
            const uint32_t r = col0 + wt;
            p.pml[row0 + r] =
                make_float2(-t.nm[r], (sum[r] + sum[RT + r]) + (sum[2 * RT + r] + sum[3 * RT + r]));
        }
        bar_sync(1, kBtSoft);  // before the next item's rows come into the same places
    }
    if (tid == 0 && (start || c.pos >= c.len)) {
        uint2 *cta = p.pcta + item;
        if (start) cta->x = blockIdx.x;
        if (c.pos >= c.len) cta->y = blockIdx.x;
    }
    if (fresh && c.left) beam_next_item(a, p, c);
}

template <typename T, int HD>
__global__ void __launch_bounds__(kBtThreads, 1)
    beam_attn_tc_kernel(const BeamAttnArgs a, const BeamAttnPlan p, const __grid_constant__ BeamMaps maps) {
    using Sm = BeamTc<HD>;
    constexpr int RT = kBtRows;
    extern __shared__ __align__(1024) uint8_t bt_sm[];
    BeamTcTail &t = *reinterpret_cast<BeamTcTail *>(bt_sm + Sm::kOffTail);
    const uint32_t warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    pdl_launch();
    BeamCursor c;
    if (!beam_first(a, p, c)) {  // the same in every thread
        pdl_wait();
        return;
    }
    if (threadIdx.x < 128) t.top[threadIdx.x] = 0;
    if (threadIdx.x == 0) {
        for (int i = 0; i < 2; ++i) {
            mbar_init(&t.kfull[i], 32);
            mbar_init(&t.vfull[i], 32);
            mbar_init(&t.kempty[i], 1);
            mbar_init(&t.vempty[i], 1);
            mbar_init(&t.sfull[i], 1);
            mbar_init(&t.sfree[i], kBtSoft / 32);
            mbar_init(&t.pfull[i], kBtSoft / 32);
            mbar_init(&t.odone[i], 1);
        }
        mbar_init(&t.ofree, kBtSoft / 32);
        mbar_init(&t.qfull, 1);
        fence_mbar_init();
    }
    if (warp == 1) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&t.tmem)), "r"(Sm::kTmem) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    bt_fence_before();
    __syncthreads();
    bt_fence_after();
    const uint32_t tmem = t.tmem;
    if (warp == 0) {
        // K of tile i + 1 before V of tile i
        BeamCursor v = c;
        uint32_t nk = 0, nv = 0;
        const bool tma = p.tma & 1;
        bool ok = true;
        auto next = [&](BeamCursor &at, uint32_t &count, const void *base, uint32_t off, const CUtensorMap *map,
                        const CUtensorMap *wide, uint64_t *full, uint64_t *empty) {
            const uint32_t s = count & 1;
            if (count >= 2) ok = mbar_wait_warp(&empty[s], (count >> 1 & 1) ^ 1, &g_beam_err, ERR_WAIT_EMPTY);
            if (!ok) return;
            const uint32_t n = bt_take(at);
            bt_copy<T, HD>(a, at, n, tma, smem_u32(bt_sm + off + s * Sm::kTile), base, map, wide, &full[s]);
            ++count;
            beam_advance(at, n);
            if (at.left && at.pos >= at.len) beam_next_item(a, p, at);
        };
        while (ok && v.left) {
            while (ok && c.left && nk <= nv + 1) next(c, nk, a.pk, 0, &maps.pk, &maps.wk, t.kfull, t.kempty);
            if (ok) next(v, nv, a.pv, Sm::kOffV, &maps.pv, &maps.wv, t.vfull, t.vempty);
        }
        // no copy is in flight when this CTA's shared memory is given back
        for (uint32_t j = 0; j < min(nk, 2u); ++j)
            mbar_wait(&t.kfull[(nk - 1 - j) & 1], (nk - 1 - j) >> 1 & 1, &g_beam_err, ERR_WAIT_DRAIN);
        for (uint32_t j = 0; j < min(nv, 2u); ++j)
            mbar_wait(&t.vfull[(nv - 1 - j) & 1], (nv - 1 - j) >> 1 & 1, &g_beam_err, ERR_WAIT_DRAIN);
    } else if (warp == 1) {
        if (lane == 0) {
            const uint32_t q = smem_u32(bt_sm + Sm::kOffQ);
            const uint32_t ids = bt_idesc<T>(RT, false), ido = bt_idesc<T>(RT, true);
            uint32_t seg = 0;
            bool ok = true;
            // S^T = K Q^T of tile i
            auto scores = [&](uint32_t i) {
                const uint32_t b = i & 1, k = smem_u32(bt_sm + b * Sm::kTile);
                bt_fence_after();
                bt_fence_proxy();
                if (ok)
#pragma unroll
                    for (int d = 0; d < HD / 16; ++d)
                        bt_mma(tmem + b * RT, bt_desc(k + (d / 4) * Sm::kSubBytes + (d % 4) * 32, 16),
                               bt_desc(q + (d / 4) * (RT * 128) + (d % 4) * 32, 16), ids, d != 0);
                bt_commit(&t.sfull[b]);
                bt_commit(&t.kempty[b]);
            };
            auto scores_ready = [&](uint32_t i) {  // its K is there and its place in tensor memory is free
                return bt_test(&t.kfull[i & 1], i >> 1 & 1) && (i < 2 || bt_test(&t.sfree[i & 1], (i >> 1 & 1) ^ 1));
            };
            auto scores_wait = [&](uint32_t i) {
                ok = mbar_wait(&t.kfull[i & 1], i >> 1 & 1, &g_beam_err, ERR_WAIT_FULL) && ok;
                if (i >= 2) ok = mbar_wait(&t.sfree[i & 1], (i >> 1 & 1) ^ 1, &g_beam_err, ERR_WAIT_EMPTY) && ok;
            };
            bool first = true;
            ok = mbar_wait(&t.qfull, 0, &g_beam_err, ERR_WAIT_FULL);
            scores_wait(0);
            scores(0);
            for (uint32_t i = 0; c.left; ++i) {
                const uint32_t n = bt_take(c), b = i & 1, ph = i >> 1 & 1;
                beam_advance(c, n);
                const bool turn = c.pos >= c.len;             // the item ends here
                bool ahead = c.left != 0 && !turn;            // the next tile's scores come first, if its K is there
                if (first && seg) ok = mbar_wait(&t.ofree, (seg - 1) & 1, &g_beam_err, ERR_WAIT_EMPTY) && ok;
                if (ahead)
                    for (uint32_t polls = 0; polls < 4096; ++polls) {
                        if (scores_ready(i + 1)) {
                            scores(i + 1);
                            ahead = false;
                            break;
                        }
                        if (bt_test(&t.pfull[b], ph)) break;
                    }
                // O^T += V^T P
                ok = mbar_wait(&t.vfull[b], ph, &g_beam_err, ERR_WAIT_FULL) && ok;
                ok = mbar_wait(&t.pfull[b], ph, &g_beam_err, ERR_WAIT_FULL) && ok;
                bt_fence_after();
                bt_fence_proxy();
                const uint32_t v = smem_u32(bt_sm + Sm::kOffV + b * Sm::kTile), ps = smem_u32(bt_sm + Sm::kOffP + b * Sm::kP);
                if (ok)
                    for (uint32_t u = 0; u < (n + kBaUnit - 1) / kBaUnit; ++u)  // (a 64-wide head: its dimensions twice)
                        bt_mma(tmem + 2 * RT, bt_desc(v + u * 2048, HD == 64 ? 0 : Sm::kSubBytes),
                               bt_desc(ps + u * 2048, Sm::kSubBytes), ido, !first || u);
                bt_commit(&t.vempty[b]);
                bt_commit(&t.odone[b]);
                first = false;
                if (turn && c.left) {
                    beam_next_item(a, p, c);
                    ++seg;
                    first = ahead = true;
                    if (c.left) ok = mbar_wait(&t.qfull, seg & 1, &g_beam_err, ERR_WAIT_FULL) && ok;
                }
                if (ahead && c.left) {
                    scores_wait(i + 1);
                    scores(i + 1);
                }
            }
        }
        __syncwarp();
    } else {
        float l[RT / 2];  // the sums of this thread's position, for half of the rows
        bool fresh = true, ok = true;
#pragma unroll 1
        for (uint32_t i = 0; c.left; ++i) bt_step<T, HD>(a, p, c, fresh, l, i, bt_sm, t, tmem, ok);
    }
    // every product is complete: the softmax waited for the last one's commit
    // (or the wait ran out after its bound)
    bt_fence_before();
    __syncthreads();
    if (warp == 1) {
        bt_fence_after();
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(Sm::kTmem) : "memory");
    }
    pdl_wait();  // the suffixes' kernel, so that what waits for this one has both
}

}  // namespace fwb
