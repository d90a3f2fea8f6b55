// beam.cu — C ABI of the beam-search operators: argument checks and launches.
#include <cuda_runtime.h>

#include <algorithm>
#include <cmath>
#include <cstdio>
#include <exception>

#include "../../include/forword_b200.h"
#include "beam_attn.cuh"
#include "beam_attn_tc.cuh"
#include "beam_reorder.cuh"
#include "beam_select.cuh"
#include "status.h"
#include "tensor_map.h"

namespace fwb {
namespace {

bool fail(const char *text) {
    set_last_error(text);
    return false;
}

bool launched(cudaError_t e, const char *who) {
    if (e == cudaSuccess) return true;
    char b[160];
    snprintf(b, sizeof b, "%s: %s", who, cudaGetErrorString(e));
    return fail(b);
}

// A kernel whose blocks may be placed while the stream's kernel before it
// ends (it waits for that one's results itself).
template <typename F, typename... A>
cudaError_t launch_after(F *fn, dim3 grid, unsigned threads, unsigned smem, unsigned cluster, cudaStream_t st, const A &...args) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = grid;
    cfg.blockDim = dim3(threads);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = st;
    cudaLaunchAttribute at[2];
    at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    at[0].val.programmaticStreamSerializationAllowed = 1;
    at[1].id = cudaLaunchAttributeClusterDimension;
    at[1].val.clusterDim.x = cluster;
    at[1].val.clusterDim.y = at[1].val.clusterDim.z = 1;
    cfg.attrs = at;
    cfg.numAttrs = cluster > 1 ? 2 : 1;
    return cudaLaunchKernelEx(&cfg, fn, args...);
}

// Dynamic shared memory past the default limit, once per kernel and device.
template <typename F>
bool opt_in(F *fn, uint32_t smem, bool (&ready)[64], const char *who) {
    int dev = 0;
    if (!launched(cudaGetDevice(&dev), who)) return false;
    if (dev < 64 && ready[dev]) return true;
    if (!launched(cudaFuncSetAttribute(fn, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem), who)) return false;
    if (dev < 64) ready[dev] = true;
    return true;
}

uint32_t elem_bytes(uint32_t type) { return type == 0 ? 4u : type == 1 || type == 30 ? 2u : 0u; }

// --- prefix attention --------------------------------------------------------
bool attn_sizes_ok(const fwb_prefix_attn_t *a) {
    if (!a) return fail("fwb_prefix_attention: null arguments");
    if (!elem_bytes(a->type)) return fail("fwb_prefix_attention: type must be 0 (F32), 1 (F16) or 30 (BF16)");
    if (!a->n_group || !a->n_beam || !a->n_query || !a->n_head || !a->n_head_kv)
        return fail("fwb_prefix_attention: zero groups, beams, query tokens or heads");
    if (a->n_head % a->n_head_kv) return fail("fwb_prefix_attention: n_head must be a multiple of n_head_kv");
    if (!a->head_dim || a->head_dim % 16 || a->head_dim > 128)
        return fail("fwb_prefix_attention: head_dim must be a multiple of 16, at most 128");
    if (a->prefix_cap > 0x7fffffffu || a->suffix_cap > 0x7fffffffu)
        return fail("fwb_prefix_attention: capacities must fit an int32");
    if (!(a->scale >= 0.f) || a->scale > 3e38f) return fail("fwb_prefix_attention: scale must be positive, or 0 for the default");
    const uint64_t rows = (uint64_t)a->n_group * a->n_beam;
    if (rows > 0xffffffu || rows * a->n_query > 0xffffffu || rows * a->n_query * a->n_head > 0x7fffffffu ||
        a->n_head > 65535)
        return fail("fwb_prefix_attention: too many sequences, tokens or heads");
    if ((uint64_t)a->n_beam * a->n_query * (a->n_head / a->n_head_kv) > 65535)
        return fail("fwb_prefix_attention: n_beam * n_query * (n_head / n_head_kv) must be at most 65535");
    return true;
}

bool attn_args(const fwb_prefix_attn_t *a, BeamAttnArgs &k) {
    if (!attn_sizes_ok(a)) return false;
    const uint64_t e = elem_bytes(a->type);
    if (!a->q || !a->out) return fail("fwb_prefix_attention: null q or out");
    if ((a->prefix_cap && (!a->prefix_k || !a->prefix_v)) || (a->suffix_cap && (!a->suffix_k || !a->suffix_v)))
        return fail("fwb_prefix_attention: null K or V");
    auto step = [&](uint64_t n, uint64_t stride) { return n > 1 ? stride * e : 0; };  // (never used where n is 1)
    const uint64_t seqs = (uint64_t)a->n_group * a->n_beam;
    uint64_t odd = (uintptr_t)a->q | step(seqs, a->q_seq_stride) | step(a->n_query, a->q_token_stride) |
                   step(a->n_head, a->q_head_stride) | (uintptr_t)a->out;
    if (a->prefix_cap)
        odd |= (uintptr_t)a->prefix_k | (uintptr_t)a->prefix_v | step(a->n_group, a->prefix_group_stride) |
               step(a->n_head_kv, a->prefix_head_stride) | step(a->prefix_cap, a->prefix_pos_stride);
    if (a->suffix_cap)
        odd |= (uintptr_t)a->suffix_k | (uintptr_t)a->suffix_v | step(seqs, a->suffix_seq_stride) |
               step(a->n_head_kv, a->suffix_head_stride) | step(a->suffix_cap, a->suffix_pos_stride);
    if (odd % 16) return fail("fwb_prefix_attention: q, K, V and out and their strides must be multiples of 16 bytes");
    if (((uintptr_t)a->lse | (uintptr_t)a->prefix_len | (uintptr_t)a->suffix_len | (uintptr_t)a->slots) % 4)
        return fail("fwb_prefix_attention: lse, lengths and slots must be 4-byte aligned");
    k = {};
    k.q = a->q; k.pk = a->prefix_k; k.pv = a->prefix_v; k.sk = a->suffix_k; k.sv = a->suffix_v;
    k.out = a->out; k.lse = a->lse;
    k.plen = a->prefix_len; k.slen = a->suffix_len; k.slots = a->slots;
    k.q_seq = a->q_seq_stride; k.q_tok = a->q_token_stride; k.q_head = a->q_head_stride;
    k.p_group = a->prefix_group_stride; k.p_head = a->prefix_head_stride; k.p_pos = a->prefix_pos_stride;
    k.s_seq = a->suffix_seq_stride; k.s_head = a->suffix_head_stride; k.s_pos = a->suffix_pos_stride;
    k.slot_seq = a->slots_stride;
    k.n_group = a->n_group; k.n_beam = a->n_beam; k.n_query = a->n_query;
    k.n_head = a->n_head; k.n_kv = a->n_head_kv; k.gq = a->n_head / a->n_head_kv; k.hd = a->head_dim;
    k.pcap = a->prefix_cap; k.scap = a->suffix_cap;
    k.scale = a->scale != 0.f ? a->scale : 1.0f / sqrtf((float)a->head_dim);
    return true;
}

uint32_t device_sms() {
    static int n[64] = {};
    int dev = 0;
    if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) return 148;
    if (!n[dev]) {
        int v = 0;
        if (cudaDeviceGetAttribute(&v, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess || v < 1) return 148;
        n[dev] = v;
    }
    return (uint32_t)n[dev];
}

// Row tiles and the workspace's layout.
struct AttnLayout {
    bool tc;            // on the 5th-generation tensor cores (beam_attn_tc.cuh)
    uint32_t prow, srow;  // rows of a prefix / suffix tile
    uint32_t ptiles, stiles, ctas, tctas, cost, tcost;  // (tctas, tcost: of the tcgen05 kernel, the others then the suffixes')
    size_t pitems, sitems, bytes;
    size_t po, so, pml, sml, pcta, scta;
};

bool attn_layout(const fwb_prefix_attn_t *a, AttnLayout &L) {
    const uint64_t gq = a->n_head / a->n_head_kv, srows = gq * a->n_query, prows = srows * a->n_beam;
    const uint32_t hd = a->head_dim <= 64 ? 64 : 128;
    // More than 64 rows over a long prefix go to the 5th-generation tensor
    // cores.  Measured (fp16, 8 KV heads of 128, one group, us for warp-level
    // products / tcgen05 over 500, 4000 and 30000 positions): 96 rows 15 / 21,
    // 24 / 24, 75 / 50; 128 rows 15 / 23, 25 / 26, 77 / 51; 256 rows 21 / 26,
    // 38 / 33, 138 / 77.  1000 positions cost the one 1 us per 64 rows and the
    // other as much per 128, and the other, two kernels, begins 5 us later.
    // (Device times of full caches.  The rule goes by the capacity, since the
    // host does not know the lengths: a cache much longer than what it holds
    // takes this path for 5 to 8 us more, by these figures.)
    const uint64_t spared = (prows + 63) / 64 - (prows + 127) / 128;
    L.tc = a->type != 0 &&
           (uint64_t)a->n_group * a->n_head_kv * a->prefix_cap * spared >= (uint64_t)36000 * device_sms() / 148;
    auto tile = [&](uint64_t rows) { return rows <= 16 ? 16u : rows <= 32 ? 32u : 64u; };
    L.prow = L.tc ? kBtRows : tile(prows);
    L.srow = tile(srows);
    L.ptiles = (uint32_t)((prows + L.prow - 1) / L.prow);
    L.stiles = (uint32_t)((srows + L.srow - 1) / L.srow);
    L.pitems = a->prefix_cap ? (size_t)a->n_group * a->n_head_kv * L.ptiles : 0;
    L.sitems = a->suffix_cap ? (size_t)a->n_group * a->n_beam * a->n_head_kv * L.stiles : 0;
    // What an item's beginning and end cost, in units.  Measured with 4 / 12 / 16:
    // 6 groups of 5 fp16 beams 40 / 32 / 32 us, 4 beams over 30000 positions 38 /
    // 30 / 31; fp32, whose units take three times as long, 30 / 31 / 32 for 4
    // beams over 8000.  Units of 64 rows take longer too: 48 beams over 500 and
    // 4000 positions 17 / 23 / - and 31 / 36 / -.  The tcgen05 kernel 20 / 40: 9
    // beams of 7 tokens 30.5 / 28.1.
    L.cost = a->type == 0 ? 4 : L.prow == 64 ? 6 : 12;
    L.tcost = 40;
    const uint64_t punits = L.pitems * ((a->prefix_cap + 15) / 16 + (L.tc ? L.tcost : L.cost)),
                   sunits = L.sitems * ((a->suffix_cap + 15) / 16 + L.cost), units = punits + sunits;
    if (L.pitems + L.sitems > 0x3fffffffu || units > 0x7fffffffu)
        return fail("fwb_prefix_attention: too many rows times positions");
    const uint64_t sms = device_sms();
    L.ctas = (uint32_t)std::max<uint64_t>(1, std::min(a->type == 0 && L.prow == 16 ? 3 * sms : 2 * sms, L.tc ? sunits : units));
    L.tctas = L.tc ? (uint32_t)std::min(sms, punits) : 0;
    size_t at = 0;
    auto take = [&](size_t n) {
        const size_t here = at;
        at += (n + 255) & ~(size_t)255;
        return here;
    };
    const size_t pslots = (L.pitems + std::max(L.ctas, L.tctas)) * L.prow, sslots = (L.sitems + L.ctas) * L.srow;
    L.po = take(pslots * hd * 4);
    L.so = take(sslots * hd * 4);
    L.pml = take(pslots * 8);
    L.sml = take(sslots * 8);
    L.pcta = take(L.pitems * 8);
    L.scta = take(L.sitems * 8);
    L.bytes = at;
    return true;
}

// A cache as a 4-D tensor; false where the copy engine does not take its
// strides (a head or group repeated by a stride of 0, say).
bool cache_map(const void *base, size_t e, uint64_t hd, uint64_t cap, uint64_t n_kv, uint64_t outer, uint64_t pos,
               uint64_t head, uint64_t out, uint32_t positions, CUtensorMap &map) {
    const auto enc = tensor_map_encoder();
    if (!cap || !enc) return false;
    const cuuint64_t dims[4] = {hd, cap, n_kv, outer};
    cuuint64_t strides[3] = {pos * e, head * e, out * e};
    for (int i = 0; i < 3; ++i) {
        if (dims[i + 1] == 1) strides[i] = hd * e;  // never used
        if (!strides[i] || strides[i] >= (cuuint64_t)1 << 40) return false;
    }
    const cuuint32_t box[4] = {(cuuint32_t)(128 / e), positions, 1, 1}, one[4] = {1, 1, 1, 1};
    const CUtensorMapDataType type = e == 4 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT32 : CU_TENSOR_MAP_DATA_TYPE_UINT16;
    return enc(&map, type, 4, const_cast<void *>(base), dims, strides, box, one, CU_TENSOR_MAP_INTERLEAVE_NONE,
               CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
               CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

// PR, SR: rows of a prefix / suffix tile.
template <typename T, int HD, int PR, int SR>
bool launch_attn(const BeamAttnArgs &k, const BeamAttnPlan &p, const BeamMaps &maps, cudaStream_t st) {
    static bool ready[64] = {};
    constexpr uint32_t smem = beam_attn_smem<T, HD, PR / 16, SR / 16>();
    if (!opt_in(beam_attn_kernel<T, HD, PR / 16, SR / 16>, smem, ready, "fwb_prefix_attention")) return false;
    beam_attn_kernel<T, HD, PR / 16, SR / 16><<<p.ctas, kBaThreads + kBaLoader, smem, st>>>(k, p, maps);
    return launched(cudaGetLastError(), "fwb_prefix_attention launch");
}

template <typename T, int HD>
bool launch_attn_tc(const BeamAttnArgs &k, const BeamAttnPlan &p, const BeamMaps &maps, cudaStream_t st) {
    static bool ready[64] = {};
    constexpr uint32_t smem = beam_tc_smem<HD>();
    static_assert(smem <= 227 * 1024, "shared memory");
    if (!opt_in(beam_attn_tc_kernel<T, HD>, smem, ready, "fwb_prefix_attention")) return false;
    return launched(launch_after(beam_attn_tc_kernel<T, HD>, dim3(p.ctas), kBtThreads, smem, 1, st, k, p, maps),
                    "fwb_prefix_attention launch");
}

template <typename T, int HD>
bool pick_attn(const BeamAttnArgs &k, const BeamAttnPlan &p, const BeamMaps &maps, cudaStream_t st) {
    switch (p.prow * 256 + p.srow) {
    case 16 * 256 + 16: return launch_attn<T, HD, 16, 16>(k, p, maps, st);
    case 32 * 256 + 16: return launch_attn<T, HD, 32, 16>(k, p, maps, st);
    case 32 * 256 + 32: return launch_attn<T, HD, 32, 32>(k, p, maps, st);
    case 64 * 256 + 16: return launch_attn<T, HD, 64, 16>(k, p, maps, st);
    case 64 * 256 + 32: return launch_attn<T, HD, 64, 32>(k, p, maps, st);
    default: return launch_attn<T, HD, 64, 64>(k, p, maps, st);
    }
}

// The kernels of a call: all parts by one, or the suffixes by that and the
// prefixes by the tcgen05 kernel; then the join.
template <typename T, int HD>
bool run_parts(const BeamAttnArgs &k, BeamAttnPlan p, const BeamMaps &maps, const AttnLayout &L, cudaStream_t st) {
    const uint32_t seqs = k.n_group * k.n_beam;
    p.part0 = L.tc ? k.n_group : 0;
    p.parts = k.n_group + seqs;
    p.cost = L.cost;
    p.ctas = L.ctas;
    if (L.tc) p.prow = p.srow;  // (its kernel has no prefix part)
    if (!pick_attn<T, HD>(k, p, maps, st)) return false;
    p.prow = L.prow;
    if constexpr (sizeof(T) == 2)
        if (L.tc) {
            p.part0 = 0;
            p.parts = k.n_group;
            p.cost = L.tcost;
            p.ctas = L.tctas;
            if (!launch_attn_tc<T, HD>(k, p, maps, st)) return false;
            p.ctas = std::max(L.ctas, L.tctas);
        }
    const uint32_t rows = seqs * k.n_query * k.n_head, sms = device_sms();
    auto join = [&](auto fn, uint32_t blocks, unsigned threads) {
        return launched(launch_after(fn, dim3(blocks), threads, 0, 1, st, k, p), "fwb_prefix_attention launch");
    };
    // (measured, all of a call on the device in us with 8 / 4 / 1 warps a row: 128 rows of 55
    // segments 30.0 / 31.2 / -, 960 of 10 - / 39.8 / 42.1, 4096 of 6 - / 142.4 / 139.4)
    if (rows <= 4 * sms) return join(beam_attn_join_kernel<T, HD, 8>, rows, kBjThreads<8>);
    if (rows <= 16 * sms) return join(beam_attn_join_kernel<T, HD, 4>, rows, kBjThreads<4>);
    return join(beam_attn_join_kernel<T, HD, 1>, (rows + 7) / 8, kBjThreads<1>);
}

template <typename T>
bool run_attn(const BeamAttnArgs &k, const AttnLayout &L, uint8_t *ws, cudaStream_t st) {
    BeamAttnPlan p{};
    p.po = reinterpret_cast<float *>(ws + L.po);
    p.so = reinterpret_cast<float *>(ws + L.so);
    p.pml = reinterpret_cast<float2 *>(ws + L.pml);
    p.sml = reinterpret_cast<float2 *>(ws + L.sml);
    p.pcta = reinterpret_cast<uint2 *>(ws + L.pcta);
    p.scta = reinterpret_cast<uint2 *>(ws + L.scta);
    p.prow = L.prow;
    p.srow = L.srow;
    p.ptiles = L.ptiles;
    p.stiles = L.stiles;
    BeamMaps maps{};
    auto prefix = [&](const void *base, uint32_t positions, CUtensorMap &m) {
        return cache_map(base, sizeof(T), k.hd, k.pcap, k.n_kv, k.n_group, k.p_pos, k.p_head, k.p_group, positions, m);
    };
    auto suffix = [&](const void *base, CUtensorMap &m) {
        return cache_map(base, sizeof(T), k.hd, k.scap, k.n_kv, k.n_group * k.n_beam, k.s_pos, k.s_head, k.s_seq,
                         kBaUnit, m);
    };
    const uint32_t whole = L.tc ? kBtKeys : sizeof(T) == 2 ? 64 : 32;
    p.tma = (prefix(k.pk, kBaUnit, maps.pk) && prefix(k.pv, kBaUnit, maps.pv) && prefix(k.pk, whole, maps.wk) &&
             prefix(k.pv, whole, maps.wv)) |
            (suffix(k.sk, maps.sk) && suffix(k.sv, maps.sv)) << 1;
    auto by = [](uint64_t d) { return d == 1 ? 0u : (uint32_t)((((uint64_t)1 << 32) + d - 1) / d); };
    p.by_gq = by(k.gq);
    p.by_query = by(k.n_query);
    return k.hd <= 64 ? run_parts<T, 64>(k, p, maps, L, st) : run_parts<T, 128>(k, p, maps, L, st);
}

// --- selection ------------------------------------------------------------------
constexpr size_t kMaxSelect = kBsMaxSelect, kMaxSelectBeams = kBsMaxBeams;

bool select_sizes_ok(uint32_t type, size_t n_group, size_t n_beam, size_t n_vocab, size_t n_select) {
    if (!elem_bytes(type)) return fail("fwb_beam_select: type must be 0 (F32), 1 (F16) or 30 (BF16)");
    if (!n_group || !n_beam || !n_vocab || !n_select)
        return fail("fwb_beam_select: zero groups, beams, tokens or selected entries");
    if (n_beam > kMaxSelectBeams || n_group > 0x7fffffffu / kMaxSelectBeams || n_vocab > 0x7fffffffu / n_beam)
        return fail("fwb_beam_select: more than 64 beams, or more than 2^31 - 1 scores in a group");
    if (n_group * n_beam > (size_t)0x7fffffff / 1025)
        return fail("fwb_beam_select: too many rows");
    if (n_select > kMaxSelect || n_select > n_beam * n_vocab)
        return fail("fwb_beam_select: n_select must be at most 128 and at most n_beam * n_vocab");
    return true;
}

// The parts of a row and the workspace's layout.
struct SelectLayout {
    uint32_t n_part, part, cap;
    size_t cand, stat, bytes;
};

// How many parts a row is read in.  More parts use more SMs; each costs about
// 7000 cycles besides its pieces (first loads, first threshold, output), and
// leaves candidates to the join (about 3000 cycles for every 512 slices of
// 32).  A piece takes a block 1800 cycles, and an SM 825 when its up to five
// blocks keep the memory busy.  The cheapest count by these figures is taken.
// Measured on the device: 256 fp32 rows of 128256 in 1 / 2 / 4 / 8 parts a row
// 45 / 38 / 40 / 45 us (2 taken); 16 bf16 rows in 2 / 5 / 8 / 16 / 32 parts 31 /
// 23 / 19 / 16 / 17 us (16); 4 fp32 rows of 32000 in 2 / 4 / 8 parts 11.8 / 9.5 /
// 8.1 us (8).
void select_layout(size_t n_group, size_t n_beam, size_t n_vocab, size_t n_select, SelectLayout &L) {
    const uint64_t rows = (uint64_t)n_group * n_beam, sms = device_sms(), piece = kBsLogits * kBsThreads;
    L.cap = (uint32_t)((2 * n_select + 16 + 31) / 32 * 32);
    uint64_t cheapest = ~0ull, count = 1;
    for (uint64_t n = 1; n <= std::min<uint64_t>(1024, (n_vocab + piece - 1) / piece); n = n < 16 ? n + 1 : n + n / 8) {
        const uint64_t pieces = ((n_vocab + n - 1) / n + piece - 1) / piece, per_sm = (rows * n + sms - 1) / sms;
        auto wave = [&](uint64_t blocks) { return blocks ? 7000 + pieces * std::max<uint64_t>(1800, 825 * blocks) : 0; };
        const uint64_t cost = per_sm / 5 * wave(5) + wave(per_sm % 5) + 3000 * ((n_beam * n * (L.cap / 32) + 511) / 512);
        if (cost < cheapest) {
            cheapest = cost;
            count = n;
        }
    }
    L.part = (uint32_t)(((n_vocab + count - 1) / count + 7) / 8 * 8);
    L.n_part = (uint32_t)((n_vocab + L.part - 1) / L.part);
    const size_t lists = rows * L.n_part;
    L.cand = 0;
    L.stat = (lists * L.cap * sizeof(float2) + 255) & ~(size_t)255;
    L.bytes = L.stat + lists * sizeof(float2);
}

template <typename T, bool VEC>
bool launch_parts(const BeamSelectArgs &k, cudaStream_t st) {
    static bool ready[64] = {};
    constexpr uint32_t smem = BeamPiece<T, VEC>::kSmem;
    if (!opt_in(beam_select_part_kernel<T, VEC>, smem, ready, "fwb_beam_select")) return false;
    beam_select_part_kernel<T, VEC><<<k.n_group * k.n_beam * k.n_part, kBsThreads, smem, st>>>(k);
    return launched(cudaGetLastError(), "fwb_beam_select launch");
}

template <typename T>
bool run_select(const BeamSelectArgs &k, cudaStream_t st) {
    // 16-byte loads when every row allows them (not row by row: rows with equal
    // logits must have equal sums)
    const bool vec = ((uintptr_t)k.logits | k.row_stride * sizeof(T)) % 16 == 0;
    if (!(vec ? launch_parts<T, true>(k, st) : launch_parts<T, false>(k, st))) return false;
    // more than one block per group when one would look at more than two
    // batches of slices: the cluster's two barriers cost about a batch
    const uint64_t batches = ((uint64_t)k.n_beam * k.n_part * (k.cap / 32) + 63) / 64;
    uint32_t cluster = 1;
    while (cluster < kBsJoinCluster && 2 * cluster < batches) cluster *= 2;
    return launched(launch_after(beam_select_join_kernel, dim3(k.n_group * cluster), kBsJoinThreads, 0, cluster, st, k),
                    "fwb_beam_select launch");
}

// --- reordering -------------------------------------------------------------------
// A state's three levels of runs, widest stride first; levels of one are left
// out.  false: its runs may overlap one another, each level not reaching past
// the stride of the next.
struct ReorderRuns {
    uint64_t n[3], stride[3], span;  // span: bytes from the first to the last
    int levels = 0;
    bool nested(uint64_t run, const size_t (&counts)[3], const size_t (&strides)[3]) {
        for (int i = 0; i < 3; ++i) {
            if (counts[i] == 1) continue;
            int at = levels++;
            for (; at > 0 && stride[at - 1] < strides[i]; --at) {
                n[at] = n[at - 1];
                stride[at] = stride[at - 1];
            }
            n[at] = counts[i];
            stride[at] = strides[i];
        }
        span = run;
        for (int i = levels - 1; i >= 0; --i) {
            uint64_t over;
            if (stride[i] < span || __builtin_mul_overflow(n[i] - 1, stride[i], &over) || over > (uint64_t)1 << 62) return false;
            span += over;
        }
        return true;
    }
    // Whether a state of the same layout, its first run `off` bytes on, shares a byte with this one.
    bool meets(int64_t off, uint64_t run, int level = 0) const {
        if (level == levels) return off < (int64_t)run && off > -(int64_t)run;
        // the two multiples of the stride around it: the smaller levels reach no further than one stride
        const int64_t st = (int64_t)stride[level], q = off / st - (off % st < 0), most = (int64_t)n[level] - 1;
        for (int64_t i = q; i <= q + 1; ++i)
            if (i >= -most && i <= most && meets(off - i * st, run, level + 1)) return true;
        return false;
    }
};

template <typename V, int NB>
bool launch_reorder(const BeamReorderArgs &k, uint64_t n, cudaStream_t st) {
    const uint64_t grid = (n + kBrThreads - 1) / kBrThreads;
    if (n + kBrThreads <= 0xffffffffu)
        beam_reorder_kernel<V, NB, uint32_t><<<(unsigned)grid, kBrThreads, 0, st>>>(k);
    else
        beam_reorder_kernel<V, NB, uint64_t><<<(unsigned)grid, kBrThreads, 0, st>>>(k);
    return launched(cudaGetLastError(), "fwb_beam_reorder launch");
}

template <typename V>
bool run_reorder(BeamReorderArgs &k, size_t run_bytes, cudaStream_t st) {
    const size_t n_col = run_bytes / sizeof(V);
    const uint64_t rows = (uint64_t)k.n_outer * k.n_inner;  // below 2^62
    if (n_col > 0xffffffffu || rows > ((uint64_t)1 << 38) / k.n_group || rows * k.n_group > ((uint64_t)1 << 38) / n_col)
        return fail("fwb_beam_reorder: state too large");
    k.n_col = (uint32_t)n_col;
    const uint64_t n = rows * k.n_group * n_col;
    if (k.n_beam <= 4) return launch_reorder<V, 4>(k, n, st);
    if (k.n_beam <= 8) return launch_reorder<V, 8>(k, n, st);
    if (k.n_beam <= 16) return launch_reorder<V, 16>(k, n, st);
    if constexpr (sizeof(V) < 16)
        if (k.n_beam > 32) return launch_reorder<V, 64>(k, n, st);
    return launch_reorder<V, 32>(k, n, st);
}

}  // namespace
}  // namespace fwb

using namespace fwb;

extern "C" {

int fwb_beam_status(void *stream) {
    uint32_t e = 0;
    try {
        if (!launched(beam_take_status(static_cast<cudaStream_t>(stream), e), "fwb_beam_status")) return -1;
    } catch (const std::exception &) {
        fail("fwb_beam_status: the lock failed");
        return -1;
    }
    if (!e) return 0;
    char b[96];
    snprintf(b, sizeof b, "fwb_beam_status: device error word 0x%x (a bounded wait in the kernel ran out)", e);
    fail(b);
    return -1;
}

size_t fwb_prefix_attention_workspace(const fwb_prefix_attn_t *a) {
    AttnLayout L;
    return attn_sizes_ok(a) && attn_layout(a, L) ? L.bytes : 0;
}

int fwb_prefix_attention_dev(const fwb_prefix_attn_t *a, void *workspace, size_t workspace_bytes, void *stream) {
    BeamAttnArgs k;
    AttnLayout L;
    if (!attn_args(a, k) || !attn_layout(a, L)) return -1;
    if (!workspace || (uintptr_t)workspace % 16 || workspace_bytes < L.bytes) {
        fail("fwb_prefix_attention: workspace missing, misaligned or smaller than fwb_prefix_attention_workspace");
        return -1;
    }
    const cudaStream_t st = static_cast<cudaStream_t>(stream);
    uint8_t *ws = static_cast<uint8_t *>(workspace);
    const bool ok = a->type == 0 ? run_attn<float>(k, L, ws, st)
                  : a->type == 1 ? run_attn<__half>(k, L, ws, st) : run_attn<__nv_bfloat16>(k, L, ws, st);
    return ok ? 0 : -1;
}

size_t fwb_beam_select_workspace(uint32_t type, size_t n_group, size_t n_beam, size_t n_vocab, size_t n_select) {
    SelectLayout L;
    if (!select_sizes_ok(type, n_group, n_beam, n_vocab, n_select)) return 0;
    select_layout(n_group, n_beam, n_vocab, n_select, L);
    return L.bytes;
}

int fwb_beam_select_dev(const void *d_logits, uint32_t type, size_t n_group, size_t n_beam, size_t n_vocab,
                        size_t row_stride, const float *d_scores, size_t n_select, float *d_out_scores,
                        int32_t *d_parent, int32_t *d_token, void *workspace, size_t workspace_bytes, void *stream) {
    if (!select_sizes_ok(type, n_group, n_beam, n_vocab, n_select)) return -1;
    if (!d_logits || !d_scores || !d_out_scores || !d_parent || !d_token) {
        fail("fwb_beam_select: null pointer");
        return -1;
    }
    if (row_stride < n_vocab) { fail("fwb_beam_select: row_stride smaller than n_vocab"); return -1; }
    if ((uintptr_t)d_logits % elem_bytes(type) ||
        ((uintptr_t)d_scores | (uintptr_t)d_out_scores | (uintptr_t)d_parent | (uintptr_t)d_token) % 4) {
        fail("fwb_beam_select: misaligned pointer");
        return -1;
    }
    SelectLayout L;
    select_layout(n_group, n_beam, n_vocab, n_select, L);
    if (!workspace || (uintptr_t)workspace % 16 || workspace_bytes < L.bytes) {
        fail("fwb_beam_select: workspace missing, misaligned or smaller than fwb_beam_select_workspace");
        return -1;
    }
    BeamSelectArgs k{};
    k.logits = d_logits; k.scores = d_scores;
    k.out_scores = d_out_scores; k.parent = d_parent; k.token = d_token;
    k.row_stride = row_stride;
    k.n_group = (uint32_t)n_group; k.n_beam = (uint32_t)n_beam; k.n_vocab = (uint32_t)n_vocab;
    k.n_select = (uint32_t)n_select;
    uint8_t *ws = static_cast<uint8_t *>(workspace);
    k.cand = reinterpret_cast<float2 *>(ws + L.cand);
    k.stat = reinterpret_cast<float2 *>(ws + L.stat);
    k.n_part = L.n_part; k.part = L.part; k.cap = L.cap;
    const cudaStream_t st = static_cast<cudaStream_t>(stream);
    const bool ok = type == 0 ? run_select<float>(k, st)
                  : type == 1 ? run_select<__half>(k, st)
                              : run_select<__nv_bfloat16>(k, st);
    return ok ? 0 : -1;
}

int fwb_beam_reorder_dev(const void *d_src, void *d_dst, const int32_t *d_parent, size_t n_outer, size_t n_group,
                         size_t n_beam, size_t n_inner, size_t run_bytes, size_t src_outer_stride,
                         size_t src_slot_stride, size_t src_inner_stride, size_t dst_outer_stride,
                         size_t dst_slot_stride, size_t dst_inner_stride, void *stream) {
    if (!d_src || !d_dst || !d_parent) { fail("fwb_beam_reorder: null pointer"); return -1; }
    if (!n_outer || !n_group || !n_beam || !n_inner || !run_bytes) { fail("fwb_beam_reorder: zero size"); return -1; }
    if (n_beam > kBrMaxBeams) { fail("fwb_beam_reorder: more than 64 beams"); return -1; }
    if (n_outer > 0x7fffffffu || n_group > 0x7fffffffu / kBrMaxBeams || n_inner > 0x7fffffffu) {
        fail("fwb_beam_reorder: sizes too large");
        return -1;
    }
    ReorderRuns to;
    if (run_bytes > (uint64_t)1 << 62 ||
        !to.nested(run_bytes, {n_outer, n_group * n_beam, n_inner}, {dst_outer_stride, dst_slot_stride, dst_inner_stride})) {
        fail("fwb_beam_reorder: the destination's runs overlap one another");
        return -1;
    }
    // the bytes from the first to the last that each side touches
    const size_t src_span = (n_outer - 1) * src_outer_stride + (n_group * n_beam - 1) * src_slot_stride +
                            (n_inner - 1) * src_inner_stride + run_bytes;
    const size_t dst_span = to.span;
    const uintptr_t s0 = (uintptr_t)d_src, d0 = (uintptr_t)d_dst;
    const bool alike = src_outer_stride == dst_outer_stride && src_slot_stride == dst_slot_stride &&
                       src_inner_stride == dst_inner_stride;
    const bool near = s0 < d0 + dst_span && d0 < s0 + src_span;
    if ((!alike && near) || (alike && near && s0 != d0 && to.meets((int64_t)(d0 - s0), run_bytes))) {
        fail("fwb_beam_reorder: source and destination overlap without being the same");
        return -1;
    }
    if ((uintptr_t)d_parent % 4) { fail("fwb_beam_reorder: misaligned parents"); return -1; }
    BeamReorderArgs k{};
    k.src = static_cast<const uint8_t *>(d_src);
    k.dst = static_cast<uint8_t *>(d_dst);
    k.parent = d_parent;
    k.src_outer = src_outer_stride; k.src_slot = src_slot_stride; k.src_inner = src_inner_stride;
    k.dst_outer = dst_outer_stride; k.dst_slot = dst_slot_stride; k.dst_inner = dst_inner_stride;
    k.n_group = (uint32_t)n_group; k.n_beam = (uint32_t)n_beam;
    k.n_outer = (uint32_t)n_outer; k.n_inner = (uint32_t)n_inner;
    const uint64_t mix = s0 | d0 | run_bytes | src_outer_stride | src_slot_stride | src_inner_stride |
                         dst_outer_stride | dst_slot_stride | dst_inner_stride;
    const cudaStream_t st = static_cast<cudaStream_t>(stream);
    // 16 bytes a column where everything allows it, 8 for the largest groups,
    // whose columns a thread could not hold otherwise
    const bool ok = mix % 16 == 0 && n_beam <= 32 ? run_reorder<uint4>(k, run_bytes, st)
                  : mix % 8 == 0                  ? run_reorder<uint2>(k, run_bytes, st)
                  : mix % 4 == 0                  ? run_reorder<uint32_t>(k, run_bytes, st)
                                                  : run_reorder<uint8_t>(k, run_bytes, st);
    return ok ? 0 : -1;
}

}  // extern "C"
