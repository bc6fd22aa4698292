/*
 * C ABI of the paged cache of ordinary attention heads (every KV head its own keys and values, a group of query heads to a KV head):
 * the pass that fills it, the attention of a decode step that reads it, and the eviction that shrinks it.  Plain pointers and sizes
 * only; all pointers are DEVICE pointers; strides are in BYTES; `stream` is a hipStream_t passed as void* (NULL = the default
 * stream); every launch returns 0, a negative MLA_ERR_* code (include/mla_attn.h) for a refused argument, or a positive hipError_t
 * value.  Nothing here allocates: scratch comes from the caller.  A *_check is the launch's own argument check alone: what it
 * returns is what the launch returns before it touches the device.
 *
 * What each entry point stands next to in the reference (paths relative to the JittorInfer tree), which builds them as separate nodes:
 *   gqa_norm_rope_launch   llm_build_norm of q and k rows, ggml_rope_ext of both (src/llama-graph-deepseek2.cpp:218-233; ggml/src/ggml.c:3413-3449)
 *                          and the cache writes of llm_build_kv_store (src/llama-graph-attn.cpp:185-217)
 *   gqa_attn_launch        ggml_flash_attn_ext over one new token with grouped heads (src/llama-graph-attn.cpp:105-120;
 *                          ggml/src/ggml-cpu/ggml-cpu.c:11914-12142)
 *   gqa_evict_launch       no counterpart: its cache only drops whole sequences or ranges of positions (src/llama-kv-cache.cpp:182-240)
 *
 * The cache.  A tensor [pages][MLA_PAGE_TOKENS rows][KV heads][width], any strides over contiguous values of a head's row, so that rows
 * may lie row by row ([page][row][head]) or head by head ([page][head][row]).  Logical row i of sequence b is row i % 128 of page
 * block_table[b * bt_stride + i / 128].  A page id outside [0, n_pages) names no memory: its rows are written nowhere and count as masked.
 */
#ifndef GQA_ATTN_H
#define GQA_ATTN_H

#include <stddef.h>
#include <stdint.h>

#include "mla_attn.h" /* MLA_TYPE_*, MLA_ERR_*, MLA_PAGE_TOKENS */

#ifdef __cplusplus
extern "C" {
#endif

typedef struct gqa_pool {
    void *  data;    /* NULL: absent */
    int64_t nb_page; /* bytes from a page, a row of a page, a head of a row to the next */
    int64_t nb_row;
    int64_t nb_head;
} gqa_pool;

/* ---- norms of queries and keys, rotation, cache write
 * For every token and head: y = x * (1 / sqrt(mean(x^2) + eps)) * weight (weight NULL: y = x), then the first n_dims values rotated by
 * the angles pos * f_i, f_i as ggml_rope_ext defines it (freq_base, freq_scale, YaRN's ext_factor / attn_factor / betas, freq_factors).
 * Angles are taken in 64 bits, so they are exact to f32 at any position; ggml_rope_ext's own f32 recurrence (mla_rope_launch) is off by
 * about pos * 2^-22 radians.  Queries go to q_dst, keys (and values, as they are) to their rows of the cache: token t of sequence
 * seq_ids[t] to row slots[t] (NULL: pos[t]); rows outside the block table, negative ones and bad pages are skipped, as the cache write
 * of include/mla_kv_write.h skips them.  Two tokens of one call that name the same row leave parts of either there; no token's k or v may lie
 * on a row that another token of the call writes. */
typedef struct gqa_norm_rope_args {
    int32_t n_tok, n_head, n_head_kv;   /* n_tok below 2^24 */
    int32_t dk, dv;          /* values per key / query head and per value head: multiples of 8, at most 256 */
    int32_t src_type;        /* of q, k, v: MLA_TYPE_F32 | MLA_TYPE_F16 | MLA_TYPE_BF16 */
    int32_t w_type;          /* of the weights: the same three */
    int32_t dst_type;        /* of q_dst: the same three */
    int32_t kv_type;         /* of the cache: MLA_TYPE_F16 | MLA_TYPE_BF16 */
    int32_t n_seq;           /* rows of the block table */
    const void * q;          /* [n_tok][n_head][dk], 16-byte aligned rows */
    int64_t q_nb1, q_nb2;    /* bytes from a head, a token to the next */
    const void * k;          /* [n_tok][n_head_kv][dk]; NULL: queries only */
    int64_t k_nb1, k_nb2;
    const void * v;          /* [n_tok][n_head_kv][dv]; NULL: no values */
    int64_t v_nb1, v_nb2;
    const void * q_weight;   /* [dk] or NULL */
    const void * k_weight;
    float eps;
    /* rotation: the fields of mla_rope_args (include/mla_front.h), in 64 bits: an angle at position 100000 shows the 25th bit of a factor */
    int32_t n_dims;          /* rotated values of a head: 0 .. dk, a multiple of 8 (mode NORM) or 16 (NEOX) */
    int32_t mode;            /* MLA_ROPE_MODE_NORM: pairs (2i, 2i + 1); MLA_ROPE_MODE_NEOX: (i, i + n_dims / 2) */
    int32_t n_ctx_orig;
    double  freq_base, freq_scale, ext_factor, attn_factor, beta_fast, beta_slow;   /* freq_base > 1 */
    const float *   freq_factors; /* [n_dims / 2] or NULL */
    const int32_t * pos;     /* [n_tok] */
    void *  q_dst;           /* [n_tok][n_head][dk]; may be q itself with the same type and strides, else apart from it */
    int64_t qd_nb1, qd_nb2;
    gqa_pool k_cache, v_cache;   /* apart from each other */
    int64_t  n_pages;
    const int32_t * block_table; /* [n_seq][bt_stride] */
    int64_t         bt_stride;
    const int32_t * seq_ids;     /* [n_tok] */
    const int32_t * slots;       /* [n_tok] row of the sequence, or NULL: pos */
} gqa_norm_rope_args;

int gqa_norm_rope_check(const gqa_norm_rope_args * args);
int gqa_norm_rope_launch(const gqa_norm_rope_args * args, void * stream);

/* ---- attention of one new token of every sequence
 * dst[b][h] = sum_i p_i v_i over the sequence's rows i (of KV head h / (n_head / n_head_kv)), p = softmax over i of
 *   s_i = scale * (q . k_i), with a soft cap c > 0 (any finite one): c * tanh(s_i / c), with a mask: + mask[b][i].
 * Rows i in [0, seq_lens[b]), with window > 0 only the last `window` of them.  A mask of -inf takes the row out whatever its key and value hold (NaN,
 * infinities); a row past the mask's end is out too.  A sequence with no row left (length 0, everything masked) gets zeros.  Lengths
 * below 0 count as 0, above the block table's room as that room.
 * weights (optional): weights[b][g][i] += sum over the query heads of KV head g of p_i, in f32 and in one order; rows outside the
 * window or the length keep their values.  dst and weights lie apart from each other, from themselves and from all that is read.
 * Supported widths (dk, dv): (64, 64), (128, 128), (192, 128), (256, 256), and (576, 0) with one KV head, without `v` and dst: the weights alone over a latent cache. */
typedef struct gqa_attn_args {
    int32_t n_seq, n_head, n_head_kv; /* n_head a multiple of n_head_kv */
    int32_t dk, dv;
    int32_t q_type;          /* MLA_TYPE_F32 (rounded to the cache's type, as ggml-cpu does) or kv_type */
    int32_t kv_type;         /* MLA_TYPE_F16 | MLA_TYPE_BF16 */
    int32_t dst_type;        /* MLA_TYPE_F32 or kv_type */
    float   scale, logit_softcap;
    int32_t window;          /* 0: every row */
    int32_t n_workgroups;    /* tuning: workgroups the rows are dealt to, 0 = choose */
    const void * q;          /* [n_seq][n_head][dk] */
    int64_t q_nb1, q_nb2;    /* bytes from a head, a sequence to the next */
    gqa_pool k, v;           /* rows 16-byte aligned, at most 8 MB apart, pages less than 4 GB */
    int64_t n_pages;
    const int32_t * block_table; /* [n_seq][bt_stride] */
    int64_t         bt_stride;
    const int32_t * seq_lens;    /* [n_seq] */
    const void * mask;       /* f16 [n_seq][mask_ne0] or NULL */
    int64_t mask_nb1, mask_ne0;
    float * weights;         /* f32 [n_seq][n_head_kv][>= bt_stride * 128] or NULL */
    int64_t w_nb1, w_nb2;    /* bytes from a KV head, a sequence to the next */
    void *  dst;             /* [n_seq][n_head][dv] */
    int64_t d_nb1, d_nb2;
    void *  workspace;       /* gqa_attn_workspace_size() bytes, 256-byte aligned */
    size_t  workspace_size;
} gqa_attn_args;

int    gqa_attn_check(const gqa_attn_args * args);          /* the workspace aside */
size_t gqa_attn_workspace_size(const gqa_attn_args * args); /* 0 for refused arguments */
int    gqa_attn_launch(const gqa_attn_args * args, void * stream);

/* ---- eviction
 * A sequence of more than n_keep rows keeps, for every KV head, its first n_sink rows, its last n_recent and, of the rest, the
 * n_keep - n_sink - n_recent of the largest weight (equal weights: the lower row; NaN counts below every number).  The rows kept move
 * up, in their order, to rows 0 .. n_keep - 1 of the same pages, keys, values and weights alike; new_lens[b] = n_keep.  Shorter
 * sequences stay as they are.  kept[b][g][j] = the row that is now row j, -1 past the new length; weights_dst past it: 0.
 * Keys keep the rotation they were written with: the next token's position goes on counting (gqa_norm_rope's pos), its row is the
 * sequence's new length (slots).  Heads keep rows of their own choice, so afterwards one row number stands for another position in every
 * head: mask and window of gqa_attn go by rows, not positions.  Pages that other sequences map too must not be evicted from
 * (mla_page_table_seq_evict refuses them); nor sequences with a page outside [0, n_pages) inside their length: nothing is read or written
 * there, so a row kept from it leaves its new place as it was, while kept, new_lens and the weights count it.  Afterwards the pages past the
 * new length are free. */
typedef struct gqa_evict_args {
    int32_t n_seq, n_head_kv;
    int32_t n_keep, n_sink, n_recent;   /* n_sink + n_recent <= n_keep.  Rows move in segments of 96 KB (24 KB where a row, a stride or an address is no multiple of
                                           16 bytes, or a row is below 32): n_seq * n_head_kv * segments of a head, K's and V's, has to stay below 2^23 */
    int32_t k_row_bytes, v_row_bytes;   /* bytes of a head's row: multiples of 4 from 8 to 16384 (any cache type, Q8_0 latent rows of 612 among them) */
    int32_t _pad;
    gqa_pool k, v;                      /* v.data NULL: keys only; else apart from each other (two halves of one row are) */
    int64_t n_pages;
    const int32_t * block_table;
    int64_t         bt_stride;
    const int32_t * seq_lens;
    const float * weights;              /* f32 [n_seq][n_head_kv][>= bt_stride * 128]; what lies past that is neither read nor written */
    int64_t w_nb1, w_nb2;
    float * weights_dst;                /* the same shape; may be `weights` itself with the same strides, else apart from it */
    int64_t wd_nb1, wd_nb2;
    int32_t * kept;                     /* [n_seq][n_head_kv][n_keep] */
    int32_t * new_lens;                 /* [n_seq]; not seq_lens itself */
    void *  workspace;                  /* gqa_evict_workspace_size() bytes, 256-byte aligned */
    size_t  workspace_size;
} gqa_evict_args;

int    gqa_evict_check(const gqa_evict_args * args);          /* the workspace aside */
size_t gqa_evict_workspace_size(const gqa_evict_args * args); /* 0 for refused arguments */
int gqa_evict_launch(const gqa_evict_args * args, void * stream);

#ifdef __cplusplus
}
#endif
#endif /* GQA_ATTN_H */
