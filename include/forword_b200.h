/*
 * forword_b200.h — C ABI of libforword_b200.so, the B200 (sm_100a) decode
 * path of forword.c.
 *
 * Plain C types only (pointers, sizes, ints).  Every function returns 0 on
 * success and -1 on failure (NULL for constructors), matching the reference's
 * error convention (transformer.c:156-164, quant_matvec.c:270-289); the
 * failure text is available from fwb_last_error().
 *
 * Threading: like the reference (single-threaded, non-reentrant), one model
 * handle must be used from one thread at a time.  Each model owns one CUDA
 * stream on its device.
 *
 * The drop-in entry points with the reference's own names
 * (transformer_init / transformer_forward / transformer_free) are in
 * forword.c_b200/shim/transformer_b200.c, which a maintainer compiles
 * together with forword.c's unchanged host C (gguf.c, model_config.c,
 * tokenizer.c, ...); it calls the fwb_* functions below.
 */
#ifndef FORWORD_B200_H
#define FORWORD_B200_H

#include <stddef.h>
#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

/* Text of the last error on this thread ("" if none).  Never NULL. */
const char *fwb_last_error(void);

/* Number of visible CUDA devices (0 when none). */
int fwb_device_count(void);

/* ------------------------------------------------------------------------
 * Quantised matrix-vector product.
 * ------------------------------------------------------------------------ */

/*
 * Replaces quant_matvec (quant_matvec.h:7-15, quant_matvec.c:263-312) with
 * the same signature and argument meaning: `weights` holds output_size rows
 * of GGUF blocks (row r at r * (input_size/32) * block_bytes), input[in] and
 * output[out] are host fp32 arrays.  The call copies weights and input to the
 * current device, runs the GEMV there and copies output back.
 * Types: 2 (Q4_0), 6 (Q5_0), 7 (Q5_1), 8 (Q8_0), 12 (Q4_K), 14 (Q6_K): the
 * reference's set (quant_matvec.c:52-62) plus GGML's Q4_0, which the
 * reference lacks.
 * Returns -1 for NULL pointers, zero sizes, an unsupported type,
 * input_size not a multiple of the block (32 values; 256 for Q4_K / Q6_K)
 * or weights_size < output_size * row bytes, like the reference.
 */
int quant_matvec(const void *weights, size_t weights_size, uint32_t ggml_type,
                 const float *input, float *output, size_t input_size,
                 size_t output_size);

/*
 * quant_matvec without any device allocation.  No counterpart in forword.c:
 * the reference's quant_matvec (quant_matvec.h:7-15) runs on the CPU; the
 * quant_matvec above keeps its signature but cudaMallocs and cudaFrees
 * device copies of weights, input and output on every call.  This variant
 * stages them in one fixed 32 MiB device array that is part of the library
 * (one per device), so a call makes no cudaMalloc, cudaFree or other
 * allocation.
 *
 * It is for callers that cannot allocate device memory at call time: a
 * process whose own memory pool (a framework's caching allocator, a serving
 * engine's KV-cache reservation) already holds the device's free memory, so
 * cudaMalloc fails or fragments it; and latency-bound loops, where the
 * implicit device-wide synchronisation of cudaFree would stall every other
 * stream of the process.
 *
 * Same arguments, element types and -1 cases as quant_matvec, and also -1,
 * with fwb_last_error() naming the bytes needed, when the call does not fit:
 * 4*input_size + the weight rows + 4*output_size + about 1 KB of alignment
 * must stay within 32 MiB (Q4_0 4096x4096 and 14336x4096 and Q8_0 4096x4096
 * fit; Q8_0 14336x4096 does not).  Synchronous, on the legacy default stream
 * of the current device.
 *
 * Set-up: the first call on each device looks up the array's device address
 * (cudaGetSymbolAddress) and sets kernel attributes; make that first call
 * before any stream capture on that device.  Only the kernel's error word
 * (the array's first 4 bytes) must be zero when the kernel starts; each call
 * zeroes it before its launch.  All calls on a device share the array: calls
 * that overlap in time on one device (from different host threads) race and
 * corrupt each other's results, so serialise them.
 */
int quant_matvec_static(const void *weights, size_t weights_size, uint32_t ggml_type,
                        const float *input, float *output, size_t input_size,
                        size_t output_size);

/*
 * Device-pointer form of quant_matvec for callers whose data already lives
 * in HBM; no reference counterpart (quant_matvec.h:7-15 is host-only).
 * d_weights must be 2-byte aligned (4-byte for Q5_1, 16-byte for Q4_K).
 * The kernel copies 16-byte aligned
 * supersets of the rows: it reads from d_weights rounded down to 16 bytes
 * (inside the same allocation unless d_weights is 16-byte aligned, as
 * cudaMalloc pointers are) up to the 16-byte boundary at or after the last
 * row, and weights_size must reach that boundary (-1 otherwise).  d_input /
 * d_output are fp32 device arrays (d_input 16-byte aligned).  `stream` is a
 * cudaStream_t (NULL = legacy default stream).  Asynchronous: returns after
 * enqueueing; quant_device_status reports a kernel-side failure.
 */
int quant_matvec_dev(const void *d_weights, size_t weights_size, uint32_t ggml_type,
                     const float *d_input, float *d_output, size_t input_size,
                     size_t output_size, void *stream);

/*
 * Status of the last quant_matvec_dev / quant_gemm_dev launch on the current
 * device after the work queued on `stream` (synchronises it): 0 if the
 * kernel completed, -1 (fwb_last_error() names the device error word) if one
 * of its bounded waits ran out and part of the output was not written.  Each
 * launch clears the word on its own stream first, so launches overlapping on
 * different streams of one device share it.  No reference counterpart: the
 * reference's quant_matvec is synchronous CPU code.
 */
int quant_device_status(void *stream);

/*
 * Batched (prompt) form of quant_matvec_dev on the tensor cores:
 * output[m * output_size + o] = sum_k W[o][k] * input[m * input_size + k] for
 * m < n_tokens (or += with accumulate != 0).  d_input_f16 holds fp16
 * activations (16-byte aligned); the products are accumulated in fp32.  This
 * is the dense contraction of a prompt's tokens sharing each weight tile, the
 * batched counterpart of linear_forward (linear.c:155-223), which the
 * reference only runs one token at a time.  Only Q4_0 (type 2) with
 * input_size a multiple of 64; other cases return -1.  Asynchronous.
 */
int quant_gemm_dev(const void *d_weights, size_t weights_size, uint32_t ggml_type, const void *d_input_f16,
                   float *d_output, size_t input_size, size_t output_size, size_t n_tokens, int accumulate,
                   void *stream);

/*
 * Dequantise n_values (a multiple of the block) from Q4_0 / Q5_0 / Q5_1 /
 * Q8_0 / Q4_K / Q6_K blocks into fp32 on the device, bit-identical to the
 * reference decoders (quant.c: q5_1_decode, q8_0_decode, q4_k_decode,
 * q6_k_decode; q5_0 as linear.c:40-56; GGML's Q4_0).
 */
int quant_dequant_dev(const void *d_weights, size_t weights_size, uint32_t ggml_type,
                      float *d_out, size_t n_values, void *stream);

/* ------------------------------------------------------------------------
 * Beam search and parallel continuations of one prompt (no reference
 * counterpart: forword.c keeps one sequence).  Sequences come in n_group
 * groups of n_beam; sequence s = group * n_beam + beam.  The operators take
 * device pointers, run on the current device, enqueue on `stream` (a
 * cudaStream_t, NULL = legacy default stream) and return without waiting;
 * they allocate nothing and may be captured into a CUDA graph.  Element
 * types are GGML's ids: 0 (F32), 1 (F16), 30 (BF16).
 * ------------------------------------------------------------------------ */

/* Arguments of fwb_prefix_attention_dev.  Strides are in elements, the
 * head_dim values of a row are contiguous; q, K and V addresses and the byte
 * strides of K and V are multiples of 16, those of q too (those of a dimension
 * of one element are not looked at). */
typedef struct fwb_prefix_attn {
    uint32_t type;                     /* of q, K, V and out: 0, 1 or 30 */
    uint32_t n_group, n_beam, n_query; /* n_query new tokens per sequence */
    uint32_t n_head, n_head_kv;        /* n_head a multiple of n_head_kv; n_beam * n_query * (their ratio) <= 65535 */
    uint32_t head_dim;                 /* a multiple of 16, at most 128 */
    uint32_t prefix_cap, suffix_cap;   /* positions that the caches hold (0: none) */
    float scale;                       /* of the scores, positive; 0 -> 1/sqrt(head_dim) */
    const void *q;                     /* [n_seq][n_query][n_head][head_dim] */
    uint64_t q_seq_stride, q_token_stride, q_head_stride;
    const void *prefix_k, *prefix_v;   /* [n_group][n_head_kv][prefix_cap][head_dim] */
    uint64_t prefix_group_stride, prefix_head_stride, prefix_pos_stride;
    const void *suffix_k, *suffix_v;   /* [n_seq][n_head_kv][suffix_cap][head_dim] */
    uint64_t suffix_seq_stride, suffix_head_stride, suffix_pos_stride;
    const int32_t *prefix_len;         /* [n_group], or NULL: prefix_cap each */
    const int32_t *suffix_len;         /* [n_seq], the new tokens included, or NULL: suffix_cap each */
    const int32_t *slots;              /* [n_seq][suffix_cap], or NULL: every position its own */
    uint64_t slots_stride;
    void *out;                         /* [n_seq][n_query][n_head][head_dim], contiguous */
    float *lse;                        /* [n_seq][n_query][n_head], or NULL */
} fwb_prefix_attn_t;

/*
 * Attention of every new token over its group's prefix (held once and read
 * once for all its beams) and its own sequence's suffix.  Token t of n_query
 * sees the prefix and the first suffix_len - (n_query - 1 - t) suffix
 * positions.  slots[s][p] = b: suffix position p of sequence s is row p of
 * sequence group * n_beam + b, the beam that computed it, so that a beam
 * step re-orders this table instead of the cache (an entry outside
 * 0..n_beam-1 counts as the sequence's own beam).  lse receives log sum exp
 * of the scaled scores.  A token that sees no position, or only ones whose
 * scores are -inf, gets out 0 and lse -inf.  Lengths are held to 0..cap; rows at and past a length are never
 * used, whatever they hold; K or V below it that is infinite or NaN reaches
 * the tokens that see its position and no others.  Scores, softmax and sums
 * are fp32, the probabilities of fp16 and bf16 calls are
 * rounded to that type for the products with V.
 * workspace: fwb_prefix_attention_workspace(a) bytes of device memory,
 * 16-byte aligned, that no other call uses meanwhile (a captured call's: at
 * every replay); its contents matter to nobody between calls.  -1 with fwb_last_error() for arguments outside the
 * above.
 */
int fwb_prefix_attention_dev(const fwb_prefix_attn_t *a, void *workspace, size_t workspace_bytes, void *stream);

/*
 * Status of the fwb_prefix_attention_dev calls on the current device since
 * the last look, after the work queued on `stream` (synchronises it): 0, or
 * -1 if one of the kernel's bounded waits ran out (its outputs are then not
 * valid); looking clears it.
 */
int fwb_beam_status(void *stream);

/* Bytes of workspace that fwb_prefix_attention_dev needs for a's type, sizes
 * and capacities (its pointers, lengths and strides are not looked at); 0
 * with fwb_last_error() for sizes that it does not take. */
size_t fwb_prefix_attention_workspace(const fwb_prefix_attn_t *a);

/*
 * Selection of a beam step: of the n_beam * n_vocab scores of a group,
 * score[w][v] = d_scores[w] + logits[w][v] - logsumexp(logits[w]), the
 * n_select largest in descending order, the lowest index w * n_vocab + v
 * first among equals: their scores, beams (0..n_beam-1) and tokens, each
 * [n_group][n_select].  d_logits holds n_group * n_beam rows of n_vocab
 * elements of `type`, row_stride elements apart; d_scores [n_group * n_beam].
 * A logit of -inf bars its token.  A row that is barred throughout, holds a
 * NaN or +inf, or has a d_scores entry that is not finite offers no
 * candidate (its scores are -inf, and still rank by index).  n_beam at most
 * 64, n_select at most 128 and at most n_beam * n_vocab, which is at most
 * 2^31 - 1.  workspace as above, of fwb_beam_select_workspace bytes.
 */
int fwb_beam_select_dev(const void *d_logits, uint32_t type, size_t n_group, size_t n_beam, size_t n_vocab,
                        size_t row_stride, const float *d_scores, size_t n_select, float *d_out_scores,
                        int32_t *d_parent, int32_t *d_token, void *workspace, size_t workspace_bytes, void *stream);
size_t fwb_beam_select_workspace(uint32_t type, size_t n_group, size_t n_beam, size_t n_vocab, size_t n_select);

/*
 * Per-beam state moved by the parents of a beam step:
 * dst[o][g * n_beam + b][i] = src[o][g * n_beam + parent[g][b]][i] for runs
 * of run_bytes bytes, o < n_outer, i < n_inner, all strides in bytes.
 * d_dst == d_src with equal strides works in place; otherwise the two must
 * not overlap: with equal strides, in no byte (one may lie in the other's
 * gaps); with others, not from first byte to last.  The destination's runs must not overlap one another: sorted,
 * each stride reaches past the runs of the smaller ones.  A parent outside 0..n_beam-1 counts as b itself.  n_beam at
 * most 64.
 */
int fwb_beam_reorder_dev(const void *d_src, void *d_dst, const int32_t *d_parent, size_t n_outer, size_t n_group,
                         size_t n_beam, size_t n_inner, size_t run_bytes, size_t src_outer_stride,
                         size_t src_slot_stride, size_t src_inner_stride, size_t dst_outer_stride,
                         size_t dst_slot_stride, size_t dst_inner_stride, void *stream);

/* ------------------------------------------------------------------------
 * Several sequences served from one cache of 4-bit pages (no reference
 * counterpart: forword.c keeps one sequence, in fp32).  As above the
 * operators take device pointers, run on the current device, enqueue on
 * `stream`, allocate nothing and may be captured into a CUDA graph.
 *
 * The cache is [n_page][n_head_kv] lines of fwb_kv4_page_bytes(head_dim,
 * page_size) bytes, 16-byte aligned.  A position's keys and values are held in
 * blocks of 32 values, each with an fp16 scale d and codes 0..15 that stand
 * for (code - 8) * d: 4.5 bits a value (head_dim is filled up to a multiple of
 * 32).  Memory that nothing was appended to may hold anything.  pages[s][i]
 * is the page that holds positions i * page_size .. of sequence s; several
 * sequences may share pages that they only read.  lengths[s] counts the
 * positions of a sequence, its new tokens included: token t of n_new[s] (at
 * most n_query; NULL: n_query each) has position lengths[s] - n_new[s] + t,
 * and the rows of tokens t >= n_new[s] of a padded batch are neither read nor
 * written.  page_size is 16, 32, 64, 128 or 256; head_dim a multiple of 16, at
 * most 128; a page table holds at most 2^30 positions, and a call at most 2^24 -
 * 1 tokens (n_seq * n_query) and 65535 heads.
 *
 * A page outside 0..n_page-1 is neither read nor written: its positions are
 * not appended, count as not seen, and read as zeros.  The same holds for
 * positions below 0, and for the append for positions past the page table or
 * the rotation's tables (a token's q_out row is then not written).  All but
 * those below 0 set an error word, which fwb_kv4_status takes.
 * ------------------------------------------------------------------------ */

/* Bytes of a page's line for one head; 0 for sizes that are not taken. */
size_t fwb_kv4_page_bytes(uint32_t head_dim, uint32_t page_size);

/* Status of the fwb_kv4 calls on the current device since the last look,
 * after the work queued on `stream` (synchronises it): 0, or -1 if one met a
 * page or position outside its tables, or if one of the attention kernel's
 * bounded waits ran out (its outputs are then not valid); looking clears it. */
int fwb_kv4_status(void *stream);

/* Arguments of fwb_kv4_append_dev.  Strides are in elements, the head_dim
 * values of a row are contiguous; addresses and byte strides of rows are
 * multiples of 16 (those of a dimension of one element are not looked at). */
typedef struct fwb_kv4_append {
    uint32_t type;                      /* of q, k, v and q_out: 0, 1 or 30 */
    uint32_t n_seq, n_query, n_head, n_head_kv, head_dim;
    uint32_t page_size, n_page, max_pages; /* max_pages: pages of a row of the table */
    uint32_t n_pos;                     /* rows of cos and sin */
    uint32_t halves;                    /* pairs (i, i + head_dim / 2) are turned, not (2i, 2i + 1) */
    const void *q;                      /* [n_seq][n_query][n_head][head_dim], or NULL (with q_out) */
    uint64_t q_seq_stride, q_token_stride, q_head_stride;
    const void *k, *v;                  /* [n_seq][n_query][n_head_kv][head_dim] */
    uint64_t k_seq_stride, k_token_stride, k_head_stride;
    uint64_t v_seq_stride, v_token_stride, v_head_stride;
    void *q_out;                        /* as q, rows of its own; q itself, or memory apart from all that is read */
    uint64_t q_out_seq_stride, q_out_token_stride, q_out_head_stride;
    void *cache;
    const int32_t *pages;               /* [n_seq][max_pages], pages_stride apart */
    uint64_t pages_stride;
    const int32_t *lengths, *n_new;     /* [n_seq] */
    const float *cos, *sin;             /* [n_pos][head_dim / 2], contiguous, 16-byte aligned; NULL: no rotation */
} fwb_kv4_append_t;

/*
 * New tokens' queries rotated by position into q_out, their keys rotated and
 * quantised, their values quantised, into the cache.  (a, b) becomes (a cos -
 * b sin, a sin + b cos) as in rope.c:28-53.  A block's scale is d = fp16(-m /
 * 8) for its value m of largest magnitude (the positive one of two), its codes
 * floor(y / d + 8.5) held to 0..15; a key's y is the fp32 value nearest to the
 * exact rotation.  Magnitudes past 524032 are held to what the largest fp16
 * scale reaches; a block with a value that is not finite reads as NaN
 * throughout.  No two tokens of a call may have the same position of the same
 * page, and no other work may use that position meanwhile.
 */
int fwb_kv4_append_dev(const fwb_kv4_append_t *a, void *stream);

/* Arguments of fwb_kv4_read_dev. */
typedef struct fwb_kv4_read {
    uint32_t type;                      /* of k and v */
    uint32_t n_seq, n, n_head_kv, head_dim;
    uint32_t page_size, n_page, max_pages;
    const void *cache;
    const int32_t *pages;
    uint64_t pages_stride;
    const int32_t *start;               /* [n_seq] */
    const int32_t *lengths;             /* [n_seq], or NULL: no limit but the page table */
    void *k, *v;                        /* [n_seq][n][n_head_kv][head_dim], contiguous */
} fwb_kv4_read_t;

/*
 * What the cache holds at positions start[s] .. start[s] + n - 1, rounded once
 * to the type (fwb_kv_read's counterpart; row order [n][n_head_kv][head_dim]).
 * Zeros below position 0 and at and past a length or the page table.
 */
int fwb_kv4_read_dev(const fwb_kv4_read_t *a, void *stream);

/* Arguments of fwb_kv4_attention_dev (strides as in fwb_kv4_append_t). */
typedef struct fwb_kv4_attn {
    uint32_t type;                      /* of q and out: 0, 1 or 30 */
    uint32_t n_seq, n_query, n_head, n_head_kv, head_dim; /* n_head a multiple of n_head_kv */
    uint32_t page_size, n_page, max_pages;
    float scale;                        /* of the scores, positive; 0 -> 1/sqrt(head_dim) */
    const void *q;                      /* [n_seq][n_query][n_head][head_dim] */
    uint64_t q_seq_stride, q_token_stride, q_head_stride;
    const void *cache;
    const int32_t *pages;               /* [n_seq][max_pages], pages_stride apart */
    uint64_t pages_stride;
    const int32_t *lengths, *n_new;     /* [n_seq]; held to 0..max_pages * page_size and 0..n_query */
    void *out;                          /* [n_seq][n_query][n_head][head_dim], contiguous */
    float *lse;                         /* [n_seq][n_query][n_head], or NULL; both apart from all that is read */
} fwb_kv4_attn_t;

/*
 * Attention of every sequence's new tokens over its pages: token t of n_new
 * sees the first lengths[s] - (n_new[s] - 1 - t) positions.  lse receives log
 * sum exp of the scaled scores.  A token that sees no position gets out 0 and
 * lse -inf; a head of it whose query holds a value that is not finite, or of
 * 2^100 or more, gets NaN, and so does one that sees a NaN key (with a NaN value,
 * the dimensions of its block); what lies past the positions that a token sees
 * reaches it in no way.  fp16 and bf16 queries are exact in the products, weighted
 * probabilities carry 16 bits; fp32 calls carry 22 and 24.
 * workspace: fwb_kv4_attention_workspace(a) bytes of device memory, 16-byte
 * aligned, that no other call uses meanwhile (a captured call's: at every
 * replay).  Its first 4096 bytes must be zeros before its first use; calls leave
 * it fit for the next one, of any sizes.  n_seq * n_query * n_head is at most 2^31 - 1, and
 * so are the query rows' tiles of 8 to 32 times the page table's tiles of 16.
 */
int fwb_kv4_attention_dev(const fwb_kv4_attn_t *a, void *workspace, size_t workspace_bytes, void *stream);

/* Bytes of workspace that fwb_kv4_attention_dev needs for a's type and sizes
 * (its pointers, lengths and strides are not looked at); 0 with
 * fwb_last_error() for sizes that it does not take. */
size_t fwb_kv4_attention_workspace(const fwb_kv4_attn_t *a);

/*
 * A token for each of n_row rows of logits (fwb_sample's counterpart for many
 * rows and given random numbers).  d_logits holds rows of n_vocab elements of
 * `type`, row_stride elements apart.  Of a row, ranked by logit and among
 * equals by the lower index, with weights exp((logit - max) / temperature):
 * the first top_k stay (0 or less: all); of these, the ones before which less
 * than top_p of their mass lies (1 or more: all); of these, the ones of weight
 * at least min_p; the first one always.  The token is the first whose running
 * mass among them exceeds d_uniform * their mass (the last of them from 1 on).
 * d_logprob (may be NULL) receives the log of its share of their mass.
 * d_temperature, d_top_k, d_top_p and d_min_p hold a value for each row; NULL:
 * 1, 0, 1 and 0.  A temperature of 0 or less takes the largest logit (log 1).
 * A logit of -inf bars its token.  A row that holds a NaN or +inf, is barred
 * throughout, or has a temperature or uniform number that is NaN gets token -1
 * and -inf.  Entries of weight below 2^-64 count as nothing, neither for top_k
 * nor in a mass; ones below 2^-32 are not drawn where they make up less than
 * 2^-24 of the mass, and a top_k or min_p that would keep some of them keeps none
 * where they make up less than 2^-20 of the mass besides the first entry's.
 * Weights carry 22 bits (fewer below 2^-8, by the rounding of an exponent to 24 bits:
 * 19 at 2^-64) and are added exactly, so a token can differ from exact arithmetic's
 * only where a limit falls within about 2^-22 of the mass of a border (2^-20 where
 * the mass is in such weights).  n_vocab at most 262144.
 */
int fwb_sample_rows_dev(const void *d_logits, uint32_t type, size_t n_row, size_t n_vocab, size_t row_stride,
                        const float *d_uniform, const float *d_temperature, const int32_t *d_top_k, const float *d_top_p,
                        const float *d_min_p, int32_t *d_token, float *d_logprob, void *stream);

/* ------------------------------------------------------------------------
 * Decode model (transformer.h:39-48 semantics).
 * ------------------------------------------------------------------------ */

typedef struct fwb_model fwb_model_t;

/*
 * transformer_init (transformer.c:14-147): open a GGUF file, derive the
 * model configuration, clamp the KV length (max_ctx 0 -> min(n_ctx, 4096);
 * max_ctx > n_ctx -> n_ctx) and upload every tensor once to HBM in its GGUF
 * byte layout.  `device` selects the CUDA device.  NULL on failure.
 */
fwb_model_t *fwb_model_open(const char *gguf_path, size_t max_ctx, int device);

/* transformer_free (transformer.c:149-165).  NULL is accepted. */
void fwb_model_close(fwb_model_t *m);

/* dims[8] = n_vocab, kv_ctx, n_embd, n_layer, n_head, n_head_kv, n_ff, head_dim */
int fwb_model_dims(const fwb_model_t *m, uint32_t *dims);

/* Quantised bytes one decode step streams (weights + norms + one embedding row). */
uint64_t fwb_model_weight_bytes(const fwb_model_t *m);

/* Time (seconds) and bytes of the tensor upload fwb_model_open did: every
 * tensor (this rank's slice under tensor parallelism) copied from the GGUF
 * mapping through pinned staging buffers by parallel host threads, with the
 * copies to the device overlapped.  No reference counterpart: the reference
 * reads its mmap on every step (tensor_data.c:25-62). */
int fwb_model_load_stats(const fwb_model_t *m, double *seconds, uint64_t *bytes);

/* Kernels one decode step launches: 1 for the persistent decode kernel
 * (default), one per phase with FWB_KERNEL_PER_PHASE=1.  -1 for NULL. */
int fwb_model_kernels_per_step(const fwb_model_t *m);

/*
 * transformer_forward (transformer.c:149-326): feed token_id at position pos
 * and write n_vocab fp32 logits to logits_host (host memory; may be NULL to
 * skip the copy).  Errors as the reference: pos >= kv_ctx or
 * token_id >= n_vocab -> -1.  A bounded wait that ran out inside the step
 * also returns -1; on one GPU the next call starts clean, under tensor
 * parallelism the model must be closed and reopened on every rank.
 */
int fwb_forward(fwb_model_t *m, uint32_t token_id, size_t pos, float *logits_host);

/*
 * Prompt processing: feed tokens[0..n) at positions pos0..pos0+n-1, as n
 * calls of fwb_forward would (main.c:145-151 feeds a prompt that way), and
 * write the logits of the last token to logits_host (may be NULL).  The first
 * n-1 tokens go through every layer together: their linear layers run as
 * dequant-GEMMs on the tensor cores (see quant_gemm_dev) with fp16
 * activations, and their K/V rows are appended to the cache; the last token
 * takes the decode step.  Models whose layer weights are not all Q4_0 (or
 * with an input width that is not a multiple of 64, or head_dim > 128, or
 * tensor parallelism) take the decode step for every token.  Set
 * FWB_PREFILL_PER_TOKEN=1 to force that path.  -1 (with fwb_last_error()) for
 * positions beyond the KV cache or token ids beyond the vocabulary.
 */
int fwb_prefill(fwb_model_t *m, const uint32_t *tokens, size_t n, size_t pos0, float *logits_host);

/* Same step, returning only the greedy next token (sampler_argmax,
 * sampler.c:28-32: the lowest index among equal maxima). */
int fwb_forward_argmax(fwb_model_t *m, uint32_t token_id, size_t pos, uint32_t *next_token);

/*
 * Greedy decode of n_steps tokens entirely on the device: step i feeds the
 * token chosen by step i-1 (first_token for i = 0) at position pos0 + i.
 * tokens_out[i] receives the token chosen by step i.
 */
int fwb_generate_greedy(fwb_model_t *m, uint32_t first_token, size_t pos0, size_t n_steps,
                        uint32_t *tokens_out);

/*
 * Sample the next token from the logits of the last step without copying
 * them to the host: main.c:176-188 with sampler.c, on the device.  The
 * repetition penalty (sampler_rep_penalty, sampler.c:86-100) is applied for
 * every entry of history[0..n_history) (prompt and generated tokens, as
 * main.c keeps them); then temperature <= 0 gives the greedy argmax
 * (sampler_argmax), otherwise temperature, softmax and top-p sampling
 * (sampler_top_p, sampler.c:46-84) with one draw of the reference's
 * xorshift64 generator, whose state *rng_state advances exactly as the
 * reference's does (only when temperature > 0).  The nucleus and the draw
 * are found by radix selection with exact fixed-point sums instead of a
 * sort of the vocabulary and the reference's fp32 running sum; the token can
 * differ from the reference's only where the draw or top_p falls within that
 * sum's rounding drift of a cumulative probability boundary (about 1e-6 of
 * the total for a nucleus of thousands of tokens, far less for peaked
 * distributions).  Under tensor parallelism every rank makes the same call (the
 * other ranks' logits are read over NVLink).  Synchronous.
 */
int fwb_sample(fwb_model_t *m, const uint32_t *history, size_t n_history, float temperature, float top_p,
               float rep_penalty, uint64_t *rng_state, uint32_t *next_token);

/*
 * Write (load) or read K/V of n positions [pos0, pos0+n) of one layer.
 * k and v are host fp32 arrays [n][n_head_kv][head_dim] — the reference's
 * kv_cache row order (kv_cache.h:13,45-51).
 */
int fwb_kv_load(fwb_model_t *m, size_t layer, size_t pos0, size_t n, const float *k,
                const float *v);
int fwb_kv_read(fwb_model_t *m, size_t layer, size_t pos0, size_t n, float *k, float *v);

/*
 * Phase timeline of the last decode step of the persistent kernel (tracing
 * aid; open the model with FWB_TRACE=1 in the environment).  GPU global timer
 * (ns) seen by CTA 0: out[2i] at the start of phase i, out[2i+1] when it
 * reaches the barrier after phase i, out[2*n_phases] at the end.  names
 * (optional) gets one NUL-terminated phase name per name_stride bytes.
 * Returns 2*n_phases + 1, or -1.
 */
int fwb_trace_read(fwb_model_t *m, uint64_t *out, size_t n, char *names, size_t name_stride);

/*
 * Barrier arrival time (GPU global timer, ns) of every CTA after every phase
 * of the last step (FWB_TRACE=1): out[phase * n_sm + cta].  Shows which CTAs
 * a barrier waits for.  Returns n_phases * n_sm, or -1.
 */
int fwb_trace_cta_read(fwb_model_t *m, uint64_t *out, size_t n);

/*
 * Timeline of every CTA's attention work item in every layer of the last
 * step (FWB_TRACE=1): out[(layer * n_sm + cta) * 8 + i], GPU global timer (ns)
 * at i = 0 start, 1 its warp 0 done with its positions, 2 partial written,
 * 3 CTA barrier passed, 4 split ticket taken, 5 item done; 0 for CTAs without
 * an item.  Clears the record.  Returns n_layer * n_sm * 8, or -1.
 */
int fwb_trace_attn_read(fwb_model_t *m, uint64_t *out, size_t n);

/*
 * Accumulated GEMV profile of the persistent kernel since the last read
 * (FWB_TRACE=1), as seen by thread 0 of each CTA:
 * out[(phase * n_sm + cta) * 8 + i] = ns spent in i = 0 input prologue,
 * 1 waiting for the first weight stage, 2 row loop, 3 tail (loop end to phase
 * end); from the phase start to 4 the first input loads landing, 5 the input
 * planes' CTA barrier; 6 from its loop end until every warp's; 7 unused.
 * Resets the counters.  Returns the number of values written, or -1.
 */
int fwb_prof_read(fwb_model_t *m, uint64_t *out, size_t n);

/* ------------------------------------------------------------------------
 * Tensor parallelism across the GPUs of one box (no reference counterpart:
 * forword.c runs on one CPU).  One process and one model handle per GPU;
 * rank r of `world` (1..8) keeps its query/KV heads, its slice of the FFN and
 * of the vocabulary, and the matching input columns of attn_output and
 * ffn_down.  After o-proj and after down-proj the ranks' partial sums are
 * added together inside the persistent decode kernel, each rank reading the
 * others' partials over NVLink from their exchange buffers; every rank ends
 * the step with the same residual stream and the same greedy token.
 * ------------------------------------------------------------------------ */

/*
 * Open rank `rank` of a `world`-rank model on CUDA device `device`: uploads
 * only this rank's slices.  n_head, n_head_kv and n_vocab must divide by
 * world, and n_ff / world and (n_head / world) * head_dim must be multiples of
 * 32.  The model can decode only after fwb_tp_connect.
 */
fwb_model_t *fwb_model_open_tp(const char *gguf_path, size_t max_ctx, int device, int rank, int world);

/* 64-byte CUDA IPC handle of this rank's exchange buffer (send it to every rank). */
int fwb_tp_handle(fwb_model_t *m, void *handle64);

/*
 * Map every rank's exchange buffer: handles = world consecutive 64-byte
 * handles in rank order (this rank's own entry is ignored).  Builds the step.
 * Every rank must then call the same forward functions with the same tokens
 * and positions; a rank that stops leaves the others waiting until their
 * bounded waits expire (an error, not a hang).  fwb_forward on any rank
 * returns all n_vocab logits (the other ranks' slices are read over NVLink);
 * fwb_logits_dev returns this rank's slice only.
 */
int fwb_tp_connect(fwb_model_t *m, const void *handles);

/*
 * Host only (no GPU): the bytes rank `rank` of `world` keeps of tensor
 * `tensor` of a GGUF file, packed row-major in GGUF block layout.  as_head:
 * the tensor is used as the LM head (vocabulary-row split).  With out NULL
 * only *out_bytes is set.
 */
int fwb_tp_shard(const char *gguf_path, const char *tensor, int as_head, int rank, int world,
                 void *out, size_t cap, size_t *out_bytes);

/*
 * Beam search: prompt[0..n) once through fwb_prefill (positions 0..n-1 of the
 * model's cache, which every beam then shares), and up to max_new tokens of
 * n_beam continuations together, with the operators above: their suffix keys
 * and values live in buffers of the call.  A continuation ends with token
 * `eos` (-1: none does) or at max_new tokens; the search ends when n_beam
 * ended ones are found and, without a length penalty, no live one can pass
 * them; live ones that are shorter than max_new then are no results.  Results
 * are sorted by the sum of log-probabilities, divided by
 * length^length_penalty (0: not divided): tokens_out [n_beam][max_new],
 * lengths_out and scores_out [n_beam] (length 0 and score -inf where there
 * are fewer).  As in fwb_prefill, and unlike the decode step, the inputs of
 * every weight product are rounded to fp16, the attention's output and the LM
 * head's input among them.  For models on one GPU whose layers and LM head are Q4_0, with
 * n + max_new <= kv_ctx and n_beam at most 64; -1 otherwise.  Synchronous.
 */
int fwb_beam_search(fwb_model_t *m, const uint32_t *prompt, size_t n, size_t n_beam, size_t max_new, int64_t eos,
                    float length_penalty, uint32_t *tokens_out, uint32_t *lengths_out, float *scores_out);

/* Device logits of the last step (n_vocab fp32) and the model's CUDA stream. */
const float *fwb_logits_dev(fwb_model_t *m);
void *fwb_stream(fwb_model_t *m);

/*
 * Page-locked host memory (cudaMallocHost) for logits_host buffers: fwb_forward
 * then copies the logits straight into it, without the staging copy a pageable
 * buffer needs.  transformer_b200.c allocates transformer_t.logits this way
 * (the reference mallocs it, transformer.c:103-115).  NULL on failure;
 * fwb_host_free accepts NULL.
 */
void *fwb_host_alloc(size_t bytes);
void fwb_host_free(void *p);

#ifdef __cplusplus
}
#endif
#endif /* FORWORD_B200_H */
