// kv4.cu — C ABI of the paged 4-bit cache: argument checks and launches.
#include <cuda_runtime.h>

#include <algorithm>
#include <cmath>
#include <exception>
#include <mutex>

#include "../../include/forword_b200.h"
#include "kv4_append.cuh"
#include "kv4_attn.cuh"
#include "kv4_attn_tc.cuh"
#include "launch.h"
#include "runs.h"

namespace fwb {
namespace {

// Until taken: kKvBad... bits, and what a bounded wait that ran out set (by
// itself: once it is set, waits give up early).
__device__ uint32_t g_kv4_err[2];

__global__ void kv4_status_kernel(uint32_t *out) {
    out[0] = atomicExch(&g_kv4_err[0], 0u);
    out[1] = atomicExch(&g_kv4_err[1], 0u);
}

uint32_t *error_word() {
    static uint32_t *at[64] = {};
    int dev = 0;
    if (!launched(cudaGetDevice(&dev), "fwb_kv4")) return nullptr;
    if (dev < 64 && at[dev]) return at[dev];
    void *p = nullptr;
    if (!launched(cudaGetSymbolAddress(&p, g_kv4_err), "fwb_kv4")) return nullptr;
    if (dev < 64) at[dev] = static_cast<uint32_t *>(p);
    return static_cast<uint32_t *>(p);
}

// The error words after the work queued on `st`, cleared in the same step.
cudaError_t take_status(cudaStream_t st, uint32_t (&word)[2]) {
    static std::mutex one;  // look at a time: they share the place that the kernel writes
    static uint32_t *place = nullptr;
    const std::lock_guard<std::mutex> lock(one);
    cudaError_t e = place ? cudaSuccess : cudaHostAlloc(&place, 2 * sizeof *place, cudaHostAllocPortable);
    if (e != cudaSuccess) return e;
    kv4_status_kernel<<<1, 1, 0, st>>>(place);
    e = cudaGetLastError();
    if (e == cudaSuccess) e = cudaStreamSynchronize(st);
    if (e == cudaSuccess)
        for (int i = 0; i < 2; ++i) word[i] = static_cast<volatile uint32_t *>(place)[i];
    return e;
}

bool refuse(const char *who, const char *what) {
    char b[200];
    snprintf(b, sizeof b, "%s: %s", who, what);
    return fail(b);
}

uint32_t log2_of(uint32_t page_size) {
    uint32_t n = 0;
    while (1u << n < page_size) ++n;
    return n;
}

bool page_ok(const char *who, uint32_t hd, uint32_t page_size) {
    if (!hd || hd % 16 || hd > 32 * kKvMaxBlocks) return refuse(who, "head_dim must be a multiple of 16, at most 128");
    if (page_size < 16 || page_size > 256 || (page_size & (page_size - 1)))
        return refuse(who, "page_size must be 16, 32, 64, 128 or 256");
    return true;
}

bool cache_ok(const char *who, uint32_t type, uint32_t n_seq, uint32_t n_tok, uint32_t n_kv, uint32_t hd, uint32_t page_size,
              uint32_t n_page, uint32_t max_pages) {
    if (!elem_bytes(type)) return refuse(who, "type must be 0 (F32), 1 (F16) or 30 (BF16)");
    if (!n_seq || !n_tok || !n_kv || !n_page || !max_pages) return refuse(who, "zero sequences, tokens, heads or pages");
    if (!page_ok(who, hd, page_size)) return false;
    if (n_page > 0x7fffffffu || (uint64_t)max_pages * page_size > 0x40000000u)
        return refuse(who, "more than 2^30 positions in a page table, or too many pages");
    if (n_kv > 65535 || n_seq > 0xffffffu || (uint64_t)n_seq * n_tok > 0xffffffu)
        return refuse(who, "too many sequences, tokens or heads");
    return true;
}

bool tables_ok(const char *who, const void *cache, const void *pages, const void *a, const void *b) {
    if (!cache || !pages || !a) return refuse(who, "null cache, pages or lengths");
    if ((uintptr_t)cache % 16) return refuse(who, "the cache must be 16-byte aligned");
    if (((uintptr_t)pages | (uintptr_t)a | (uintptr_t)b) % 4) return refuse(who, "tables and lengths must be 4-byte aligned");
    return true;
}

// Rows [n_seq][n_tok][heads][head_dim] whose addresses and byte strides are
// multiples of 16 (those of a dimension of one element are not looked at).
bool rows_ok(const char *who, uint32_t type, uint32_t n_seq, uint32_t n_tok, uint32_t heads, const Kv4Rows &r) {
    const uint64_t e = elem_bytes(type);
    auto step = [&](uint64_t n, uint64_t stride) { return n > 1 ? stride * e : 0; };
    if (((uintptr_t)r.p | step(n_seq, r.seq) | step(n_tok, r.tok) | step(heads, r.head)) % 16)
        return refuse(who, "rows and their strides must be multiples of 16 bytes");
    return true;
}

// Rotated queries: rows of their own that do not lie over one another, and the
// queries' own memory or memory apart from it.
bool rows_out_ok(const char *who, uint64_t run, const size_t (&n)[3], const Kv4Rows &from, const Kv4Rows &to, uint64_t e) {
    const size_t in[3] = {from.seq * e, from.tok * e, from.head * e}, out[3] = {to.seq * e, to.tok * e, to.head * e};
    Runs runs;
    if (!runs.nested(run, n, out)) return refuse(who, "q_out's rows overlap one another");
    bool alike = true;
    uint64_t span = run;  // of the queries
    for (int i = 0; i < 3; ++i) {
        if (n[i] == 1) continue;
        alike = alike && in[i] == out[i];
        uint64_t over;
        if (__builtin_mul_overflow(n[i] - 1, in[i], &over) || __builtin_add_overflow(span, over, &span)) span = UINT64_MAX / 2;
    }
    const uint64_t at = (uintptr_t)from.p, to_at = (uintptr_t)to.p;
    const bool near = to_at < at ? at - to_at < runs.span : to_at - at < span;
    if (near && (!alike || (at != to_at && runs.meets((int64_t)(to_at - at), run))))
        return refuse(who, "q_out must be q itself or memory apart from it");
    return true;
}

template <typename T>
bool run_append(const Kv4AppendArgs &k, bool halves, dim3 grid, cudaStream_t st) {
    const auto fn = !k.cos ? kv4_append_kernel<T, kKpNone> : halves ? kv4_append_kernel<T, kKpHalves> : kv4_append_kernel<T, kKpNeighbours>;
    return launched(launch_after(fn, grid, kKpThreads, 0, 1, st, k), "fwb_kv4_append launch");
}

// --- attention ---------------------------------------------------------------
constexpr const char *kAttn = "fwb_kv4_attention";

bool attn_sizes_ok(const fwb_kv4_attn_t *a) {
    if (!a) return refuse(kAttn, "null arguments");
    if (!cache_ok(kAttn, a->type, a->n_seq, a->n_query, a->n_head_kv, a->head_dim, a->page_size, a->n_page, a->max_pages)) return false;
    if (!a->n_head || a->n_head % a->n_head_kv) return refuse(kAttn, "n_head must be a multiple of n_head_kv");
    if (!(a->scale >= 0.f) || a->scale > 3e38f) return refuse(kAttn, "scale must be positive, or 0 for the default");
    if (a->n_head > 65535 || (uint64_t)a->n_seq * a->n_query * a->n_head > 0x7fffffffu)
        return refuse(kAttn, "too many sequences, tokens or heads");
    return true;
}

struct AttnLayout {
    bool tc;                              // on the 5th-generation tensor cores (kv4_attn_tc.cuh)
    uint32_t nt, nb, rows, rtiles, ctas;  // column tiles of 8 rows, blocks of a row, rows of a tile, row tiles, CTAs
    size_t po, pml, ticket, bytes;
};

bool attn_layout(const fwb_kv4_attn_t *a, AttnLayout &L) {
    const uint64_t rows = (uint64_t)a->n_query * (a->n_head / a->n_head_kv);
    L.nt = rows <= 8 ? 1 : rows <= 16 ? 2 : 4;
    L.nb = kv4_blocks(a->head_dim);
    // More rows than half a tile of the tcgen05 kernel, and tiles for three
    // quarters of the SMs (their items are better left whole: a part is 64 KB).
    // Measured, us for warp-level products / tcgen05 (fp16, 8 KV heads of 128, 4
    // query heads each): 512 tokens at 8191 positions (128 tiles) 420 / 244, at 512
    // 63 / 28; 16 sequences of 1000 positions with 16, 32, 64 tokens (128, 128, 256
    // tiles) 55 / 42, 94 / 43, 167 / 82, 12 with 32 (96) 76 / 41; of one sequence 32, 64,
    // 128, 256 tokens at 8191 (8, 16, 32, 64 tiles) 47 / 215, 70 / 218, 120 / 217, 222 / 222.
    // (Between half and three quarters of the SMs equal lengths would gain, unequal
    // ones, whose longest item is one CTA's, lose.)
    const uint64_t tiles = (uint64_t)a->n_seq * a->n_head_kv * ((rows + kKtRows - 1) / kKtRows);
    L.tc = a->type != 0 && (L.nb == 2 || L.nb == 4) && rows >= kKtRows / 2 && 4 * tiles >= 3 * (uint64_t)device_sms();
    L.rows = L.tc ? kKtRows : 8 * L.nt;
    L.rtiles = (uint32_t)((rows + L.rows - 1) / L.rows);
    const uint64_t units = (uint64_t)a->n_seq * L.rtiles * a->n_head_kv * ((uint64_t)a->max_pages * a->page_size / kKvTile + 64);
    if (units > 0x7fffffffu) return refuse(kAttn, "too many rows times positions");
    L.ctas = device_sms() * (!L.tc && L.nt <= 2 ? 2 : 1);
    size_t at = 0;
    auto take = [&](size_t n) {
        const size_t here = at;
        at += (n + 255) & ~(size_t)255;
        return here;
    };
    L.ticket = take(device_sms() * 2 * 4);  // (in the same place for all sizes: it is zero between calls)
    L.pml = take((size_t)2 * L.ctas * L.rows * 8);
    L.po = take((size_t)2 * L.ctas * L.rows * 32 * L.nb * 4);
    L.bytes = at;
    return true;
}

template <bool SPLIT, int NB, int NT>
bool launch_attn(const Kv4AttnArgs &k, uint32_t ctas, cudaStream_t st) {
    static bool ready[64] = {};
    constexpr uint32_t smem = KaSmem<SPLIT, NB, NT>::kBytes;
    if (!opt_in(kv4_attn_kernel<SPLIT, NB, NT>, smem, ready, kAttn)) return false;
    return launched(launch_after(kv4_attn_kernel<SPLIT, NB, NT>, dim3(ctas), kKaThreads, smem, 1, st, k), kAttn);
}

template <typename T, int NB>
bool launch_attn_tc(const Kv4AttnArgs &k, uint32_t ctas, cudaStream_t st) {
    static bool ready[64] = {};
    constexpr uint32_t smem = kt_smem<NB>();
    static_assert(smem <= 227 * 1024, "shared memory");
    if (!opt_in(kv4_attn_tc_kernel<T, NB>, smem, ready, kAttn)) return false;
    return launched(launch_after(kv4_attn_tc_kernel<T, NB>, dim3(ctas), kKtThreads, smem, 1, st, k), kAttn);
}

template <bool SPLIT, int NB>
bool pick_rows(const Kv4AttnArgs &k, const AttnLayout &L, cudaStream_t st) {
    return L.nt == 1 ? launch_attn<SPLIT, NB, 1>(k, L.ctas, st)
         : L.nt == 2 ? launch_attn<SPLIT, NB, 2>(k, L.ctas, st) : launch_attn<SPLIT, NB, 4>(k, L.ctas, st);
}

template <bool SPLIT>
bool pick_blocks(const Kv4AttnArgs &k, const AttnLayout &L, cudaStream_t st) {
    switch (L.nb) {
    case 1: return pick_rows<SPLIT, 1>(k, L, st);
    case 2: return pick_rows<SPLIT, 2>(k, L, st);
    case 3: return pick_rows<SPLIT, 3>(k, L, st);
    default: return pick_rows<SPLIT, 4>(k, L, st);
    }
}

}  // namespace
}  // namespace fwb

using namespace fwb;

extern "C" {

size_t fwb_kv4_page_bytes(uint32_t head_dim, uint32_t page_size) {
    return page_ok("fwb_kv4_page_bytes", head_dim, page_size) ? (size_t)page_size / kKvTile * kv4_tile(kv4_blocks(head_dim)) : 0;
}

int fwb_kv4_status(void *stream) {
    uint32_t e[2] = {0, 0};
    try {
        if (!launched(take_status(static_cast<cudaStream_t>(stream), e), "fwb_kv4_status")) return -1;
    } catch (const std::exception &) {
        fail("fwb_kv4_status: the lock failed");
        return -1;
    }
    if (!e[0] && !e[1]) return 0;
    char b[200];
    snprintf(b, sizeof b, "fwb_kv4_status:%s%s%s", e[0] & kKvBadPage ? " a page outside the cache" : "",
             e[0] & kKvBadPosition ? " a position past the page table or the rotation's tables" : "",
             e[1] ? " a bounded wait in the kernel ran out" : "");
    fail(b);
    return -1;
}

int fwb_kv4_append_dev(const fwb_kv4_append_t *a, void *stream) {
    constexpr const char *who = "fwb_kv4_append";
    if (!a) { refuse(who, "null arguments"); return -1; }
    if (!cache_ok(who, a->type, a->n_seq, a->n_query, a->n_head_kv, a->head_dim, a->page_size, a->n_page, a->max_pages) ||
        !tables_ok(who, a->cache, a->pages, a->lengths, a->n_new))
        return -1;
    if (!a->k || !a->v || !a->q != !a->q_out || (a->q && !a->n_head)) {
        refuse(who, "null k or v, or only one of q and q_out");
        return -1;
    }
    if (!a->cos != !a->sin || (a->cos && !a->n_pos) || ((uintptr_t)a->cos | (uintptr_t)a->sin) % 16) {
        refuse(who, "cos and sin must both be given, 16-byte aligned, with n_pos rows, or both be null");
        return -1;
    }
    const uint32_t heads = a->q ? a->n_head : 0;
    Kv4AppendArgs k{};
    k.q = {a->q, a->q_seq_stride, a->q_token_stride, a->q_head_stride};
    k.k = {a->k, a->k_seq_stride, a->k_token_stride, a->k_head_stride};
    k.v = {a->v, a->v_seq_stride, a->v_token_stride, a->v_head_stride};
    k.q_out = {a->q_out, a->q_out_seq_stride, a->q_out_token_stride, a->q_out_head_stride};
    if (!rows_ok(who, a->type, a->n_seq, a->n_query, a->n_head_kv, k.k) || !rows_ok(who, a->type, a->n_seq, a->n_query, a->n_head_kv, k.v) ||
        (heads && (!rows_ok(who, a->type, a->n_seq, a->n_query, heads, k.q) || !rows_ok(who, a->type, a->n_seq, a->n_query, heads, k.q_out))))
        return -1;
    if (heads > 65535) { refuse(who, "too many heads"); return -1; }
    const uint64_t e = elem_bytes(a->type);
    if (heads && !rows_out_ok(who, a->head_dim * e, {a->n_seq, a->n_query, heads}, k.q, k.q_out, e)) return -1;
    k.cache = static_cast<uint8_t *>(a->cache);
    k.pages = a->pages; k.len = a->lengths; k.n_new = a->n_new;
    k.cos = a->cos; k.sin = a->sin;
    k.pages_seq = a->pages_stride;
    k.n_seq = a->n_seq; k.n_query = a->n_query; k.n_head = heads; k.n_kv = a->n_head_kv; k.hd = a->head_dim;
    k.page_log2 = log2_of(a->page_size); k.n_page = a->n_page; k.max_pages = a->max_pages; k.n_pos = a->n_pos;
    auto by = [](uint64_t d) { return d == 1 ? 0u : (uint32_t)((((uint64_t)1 << 32) + d - 1) / d); };
    const uint32_t pairs = a->head_dim * elem_bytes(a->type) / 32;  // of 16-byte chunks in a query row
    k.by_part = by(pairs);
    k.by_blocks = by(kv4_blocks(a->head_dim));
    if (!(k.err = error_word())) return -1;
    // Blocks of a token: one where tokens fill the device; few tokens are dealt out finer.
    const uint32_t tokens = a->n_seq * a->n_query, most = std::max(heads * pairs, 2 * a->n_head_kv * kv4_blocks(a->head_dim) * 4),
                   parts = std::min((most + kKpThreads - 1) / kKpThreads, std::max(1u, 4 * device_sms() / tokens));
    const cudaStream_t st = static_cast<cudaStream_t>(stream);
    const dim3 grid(tokens, parts);
    const bool ok = a->type == 0 ? run_append<float>(k, a->halves != 0, grid, st)
                  : a->type == 1 ? run_append<__half>(k, a->halves != 0, grid, st)
                                 : run_append<__nv_bfloat16>(k, a->halves != 0, grid, st);
    return ok ? 0 : -1;
}

int fwb_kv4_read_dev(const fwb_kv4_read_t *a, void *stream) {
    constexpr const char *who = "fwb_kv4_read";
    if (!a) { refuse(who, "null arguments"); return -1; }
    if (!cache_ok(who, a->type, a->n_seq, a->n, a->n_head_kv, a->head_dim, a->page_size, a->n_page, a->max_pages) ||
        !tables_ok(who, a->cache, a->pages, a->start, a->lengths))
        return -1;
    if (!a->k || !a->v || ((uintptr_t)a->k | (uintptr_t)a->v) % 16) { refuse(who, "null or misaligned k or v"); return -1; }
    const uint64_t lanes = (uint64_t)a->n_seq * a->n * 2 * a->n_head_kv * (a->head_dim / 4);
    if (lanes > 0xffffff00u) { refuse(who, "too many positions or heads"); return -1; }
    Kv4ReadArgs k{};
    k.cache = static_cast<const uint8_t *>(a->cache);
    k.pages = a->pages; k.start = a->start; k.len = a->lengths;
    k.k = a->k; k.v = a->v;
    k.pages_seq = a->pages_stride;
    k.type = a->type; k.n_seq = a->n_seq; k.n = a->n; k.n_kv = a->n_head_kv; k.hd = a->head_dim;
    k.page_log2 = log2_of(a->page_size); k.n_page = a->n_page; k.max_pages = a->max_pages;
    if (!(k.err = error_word())) return -1;
    const uint32_t blocks = (uint32_t)((lanes + kKpThreads - 1) / kKpThreads);
    return launched(launch_after(kv4_read_kernel, dim3(blocks), kKpThreads, 0, 1, static_cast<cudaStream_t>(stream), k), who) ? 0 : -1;
}

size_t fwb_kv4_attention_workspace(const fwb_kv4_attn_t *a) {
    AttnLayout L;
    return attn_sizes_ok(a) && attn_layout(a, L) ? L.bytes : 0;
}

int fwb_kv4_attention_dev(const fwb_kv4_attn_t *a, void *workspace, size_t workspace_bytes, void *stream) {
    AttnLayout L;
    if (!attn_sizes_ok(a) || !attn_layout(a, L) || !tables_ok(kAttn, a->cache, a->pages, a->lengths, a->n_new)) return -1;
    if (!a->q || !a->out) { refuse(kAttn, "null q or out"); return -1; }
    if (!rows_ok(kAttn, a->type, a->n_seq, a->n_query, a->n_head, {a->q, a->q_seq_stride, a->q_token_stride, a->q_head_stride})) return -1;
    if ((uintptr_t)a->out % 16 || (uintptr_t)a->lse % 4) { refuse(kAttn, "out must be 16-byte and lse 4-byte aligned"); return -1; }
    if (!workspace || (uintptr_t)workspace % 16 || workspace_bytes < L.bytes) {
        refuse(kAttn, "workspace missing, misaligned or smaller than fwb_kv4_attention_workspace");
        return -1;
    }
    uint8_t *ws = static_cast<uint8_t *>(workspace);
    Kv4AttnArgs k{};
    k.q = a->q; k.cache = static_cast<const uint8_t *>(a->cache);
    k.pages = a->pages; k.len = a->lengths; k.n_new = a->n_new;
    k.out = a->out; k.lse = a->lse;
    k.q_seq = a->q_seq_stride; k.q_tok = a->q_token_stride; k.q_head = a->q_head_stride; k.pages_seq = a->pages_stride;
    k.type = a->type; k.n_seq = a->n_seq; k.n_query = a->n_query; k.n_head = a->n_head; k.n_kv = a->n_head_kv;
    k.gq = a->n_head / a->n_head_kv; k.hd = a->head_dim;
    k.tpp_log2 = log2_of(a->page_size) - 4; k.n_page = a->n_page; k.max_pages = a->max_pages;
    k.rtiles = L.rtiles;
    // How the line is cut, in pairs of tiles.  Measured (us on the device): an
    // item's ends counted as 8 / 16 / 24 / 32 pairs, 64 sequences of up to 8191
    // 110 / 96 / 93 / 95; parts of at least 16 / 24 / 40 pairs, one sequence of
    // 4000 positions 12.7 / 14.8 / 16.8, of 16000 17.4 / 18.9 / 17.6; items of up
    // to 48 pairs left whole where there is a CTA for each: 1000 positions 12.2,
    // cut 12.6 (2000: whole 17.7, cut 13.2).
    k.cost = 24;
    k.snap = 8;
    k.least = 16;
    k.whole = 48;
    k.scale = a->scale != 0.f ? a->scale : 1.0f / sqrtf((float)a->head_dim);
    k.po = reinterpret_cast<float *>(ws + L.po);
    k.pml = reinterpret_cast<float2 *>(ws + L.pml);
    k.ticket = reinterpret_cast<uint32_t *>(ws + L.ticket);
    if (!(k.err = error_word())) return -1;
    k.wait_err = k.err + 1;
    const cudaStream_t st = static_cast<cudaStream_t>(stream);
    if (L.tc) {
        // in tiles of 64 positions; items with a CTA each are left whole, others cut
        // only past 16 tiles of their ends
        k.cost = 12;
        k.snap = 16;
        k.least = 32;
        k.whole = 0x3fffffff;
        const bool ok = a->type == 1 ? (L.nb == 4 ? launch_attn_tc<__half, 4>(k, L.ctas, st) : launch_attn_tc<__half, 2>(k, L.ctas, st))
                                     : (L.nb == 4 ? launch_attn_tc<__nv_bfloat16, 4>(k, L.ctas, st) : launch_attn_tc<__nv_bfloat16, 2>(k, L.ctas, st));
        return ok ? 0 : -1;
    }
    return (a->type == 0 ? pick_blocks<true>(k, L, st) : pick_blocks<false>(k, L, st)) ? 0 : -1;
}

}  // extern "C"
