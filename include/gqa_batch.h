/*
 * C ABI of attention in which a row of keys serves many queries, for layers that keep keys and values per head: many new tokens of a sequence over its
 * pages (a prompt, a chunk of one, draft tokens to verify), a decoder's tokens over an encoder's states, one new token of sequences
 * that share their first rows.  Plain pointers and sizes only; all pointers are DEVICE pointers; strides are in BYTES; `stream` is a hipStream_t passed as
 * void* (NULL = the default stream); every launch returns 0, a negative MLA_ERR_* code (include/mla_attn.h) for a refused argument, or a positive
 * hipError_t value.  Nothing here allocates: scratch comes from the caller.  A *_check is the launch's own argument check alone (the workspace aside): what it
 * returns is what the launch returns before it touches the device.
 *
 * What each entry point stands next to in the reference (paths relative to the JittorInfer tree):
 *   gqa_prompt_attn_launch   ggml_flash_attn_ext of a batch of tokens with a causal mask, grouped heads (src/llama-graph-attn.cpp:105-120;
 *                            ggml/src/ggml-cpu/ggml-cpu.c:11914-12142); the mask of src/llama-context.cpp:354-404 is the causal rule itself
 *   gqa_cross_attn_launch    the same node with a key length of its own and no causal mask
 *   gqa_prefix_attn_launch   no counterpart: its sequences may share cells (llama_kv_cache_seq_cp, src/llama-kv-cache.cpp:242-283), which it reads for
 *                            every query of the batch under one mask
 *
 * All three: out[t][h] = sum_i p_i v_i over the rows i that token t sees (of KV head h / (n_head / n_head_kv)), p = softmax over i of
 *   s_i = scale * (q . k_i), with a soft cap c > 0 (any finite one): c * tanh(s_i / c), with a mask: + mask[b][i] of the token's sequence b.
 * A mask of -inf takes the row out whatever its key and value hold (NaN, infinities), and so do all rules of what a token sees; a row past the mask's end is out
 * too.  A token that sees no row gets zeros.  Queries, keys, values and results are of one 16-bit type; scores, maxima and sums are f32, the
 * weights p are rounded to that type (relative to a reference near the row's maximum) for the second product, as the result is after it.  A mask's number is where
 * a score's sum begins: a score is off by up to 2^-13 (bf16: 2^-10) of log2 units for it, or by half a step of the score where it is too large for that.
 * Supported widths (dk, dv): (64, 64), (128, 128), (192, 128), (256, 256).
 * The result lies apart from all that is read.
 */
#ifndef GQA_BATCH_H
#define GQA_BATCH_H

#include <stddef.h>
#include <stdint.h>

#include "gqa_attn.h" /* gqa_pool, MLA_TYPE_*, MLA_ERR_*, MLA_PAGE_TOKENS */

#ifdef __cplusplus
extern "C" {
#endif

/* ---- many new tokens of every sequence over a paged cache
 * Sequence b has the tokens q_starts[b] .. q_starts[b + 1] - 1 of q (q_starts NULL: n_tok / n_seq each, in order), whose keys and values are the last rows of its
 * cache already: token j of its n sees the rows i <= seq_lens[b] - n + j (causal) or all i < seq_lens[b], with window > 0 only the last
 * `window` of those.  Numbers in q_starts are taken to lie in [0, n_tok] and never fall; tokens outside [q_starts[0], q_starts[n_seq]) keep what dst holds.  Lengths below 0
 * count as 0, above the block table's room as that room.  A page id outside [0, n_pages) names no memory: its rows count as masked. */
typedef struct gqa_prompt_attn_args {
    int32_t n_tok, n_seq, n_head, n_head_kv; /* n_head a multiple of n_head_kv; n_tok * n_head below 2^31 */
    int32_t dk, dv;
    int32_t type;            /* of q, the cache and dst: MLA_TYPE_F16 | MLA_TYPE_BF16 */
    int32_t causal;          /* 0: every token sees its sequence's rows */
    float   scale, logit_softcap;
    int32_t window;          /* 0: no window */
    int32_t n_workgroups;    /* tuning: workgroups the work is dealt to, 0 = choose */
    const void * q;          /* [n_tok][n_head][dk], rows 16-byte aligned */
    int64_t q_nb1, q_nb2;    /* bytes from a head, a token to the next */
    const int32_t * q_starts; /* [n_seq + 1] or NULL */
    gqa_pool k, v;           /* rows 16-byte aligned, at most 8 MB apart, pages less than 4 GB */
    int64_t n_pages;
    const int32_t * block_table; /* [n_seq][bt_stride] */
    int64_t         bt_stride;
    const int32_t * seq_lens;    /* [n_seq] rows, the new ones among them */
    const void * mask;       /* f16 [n_seq][mask_ne0] or NULL */
    int64_t mask_nb1, mask_ne0;
    void *  dst;             /* [n_tok][n_head][dv], rows 8-byte aligned */
    int64_t d_nb1, d_nb2;
    void *  workspace;       /* gqa_prompt_attn_workspace_size() bytes, 256-byte aligned */
    size_t  workspace_size;
} gqa_prompt_attn_args;

int    gqa_prompt_attn_check(const gqa_prompt_attn_args * args);
size_t gqa_prompt_attn_workspace_size(const gqa_prompt_attn_args * args); /* 0 for refused arguments */
int    gqa_prompt_attn_launch(const gqa_prompt_attn_args * args, void * stream);

/* ---- a decoder's tokens over an encoder's states
 * The states of sequence b are the rows kv_starts[b] .. (kv_starts given), or 0 .. n_kv - 1 of the sequence's own part of k and v (k.nb_page bytes from a sequence to the
 * next; 0 with kv_starts); it has kv_lens[b] of them (kv_lens given), else kv_starts[b + 1] - kv_starts[b], else n_kv.  Lengths below 0 count as 0,
 * those that pass n_kv end there, and a start outside [0, n_kv] has no states.  Tokens and q_starts are those of gqa_prompt_attn; every token sees every state. */
typedef struct gqa_cross_attn_args {
    int32_t n_tok, n_seq, n_head, n_head_kv;
    int32_t dk, dv;
    int32_t type;
    int32_t n_workgroups;
    float   scale, logit_softcap;
    const void * q;
    int64_t q_nb1, q_nb2;
    const int32_t * q_starts; /* [n_seq + 1] or NULL */
    gqa_pool k, v;           /* nb_page: bytes from a sequence to the next; rows 16-byte aligned, at most 8 MB apart */
    int64_t n_kv;            /* rows of a sequence's part, or of the whole with kv_starts: below 2^30 */
    const int32_t * kv_starts; /* [n_seq + 1] ([n_seq] with kv_lens) or NULL */
    const int32_t * kv_lens;   /* [n_seq] or NULL */
    const void * mask;       /* f16 [n_seq][mask_ne0], by state of the sequence, or NULL */
    int64_t mask_nb1, mask_ne0;
    void *  dst;
    int64_t d_nb1, d_nb2;
    void *  workspace;
    size_t  workspace_size;
} gqa_cross_attn_args;

int    gqa_cross_attn_check(const gqa_cross_attn_args * args);
size_t gqa_cross_attn_workspace_size(const gqa_cross_attn_args * args);
int    gqa_cross_attn_launch(const gqa_cross_attn_args * args, void * stream);

/* ---- one new token of every sequence, where sequences share their first rows
 * What gqa_attn (include/gqa_attn.h) answers, with the shared rows read once a group.  Group g is the sequences prefix_starts[g] .. prefix_starts[g + 1] - 1 of the batch, side
 * by side; their first prefix_lens[g] rows hold the same keys and values, and are read through the block table of the first of them (rows of a page that is not
 * shared whole, too: that table names all of the prefix's pages, whatever the length of the first) or, where the table has room for so few rows that reading them once does not
 * pay, or there are as many groups as sequences (and n_workgroups is 0), through each one's own.  A sequence
 * shorter than its group's prefix sees what it has of it; sequences outside [prefix_starts[0], prefix_starts[n_prefix]) share nothing.  Numbers in prefix_starts are
 * taken to lie in [0, n_seq] and never fall; lengths of prefixes count as seq_lens do.  Rows that are read through a sequence's own table are gqa_attn's in all (weights in several parts,
 * as precise as f32; a result that an infinite value makes infinite may be NaN there).
 */
typedef struct gqa_prefix_attn_args {
    int32_t n_seq, n_prefix, n_head, n_head_kv;
    int32_t dk, dv;
    int32_t type;
    int32_t n_workgroups;
    float   scale, logit_softcap;
    const void * q;          /* [n_seq][n_head][dk] */
    int64_t q_nb1, q_nb2;
    gqa_pool k, v;           /* rows 16-byte aligned, at most 8 MB apart, pages less than 4 GB */
    int64_t n_pages;
    const int32_t * block_table;   /* [n_seq][bt_stride] */
    int64_t         bt_stride;
    const int32_t * seq_lens;      /* [n_seq] rows, the shared ones among them */
    const int32_t * prefix_starts; /* [n_prefix + 1] */
    const int32_t * prefix_lens;   /* [n_prefix] */
    const void * mask;       /* f16 [n_seq][mask_ne0] or NULL */
    int64_t mask_nb1, mask_ne0;
    void *  dst;             /* [n_seq][n_head][dv] */
    int64_t d_nb1, d_nb2;
    void *  workspace;
    size_t  workspace_size;
} gqa_prefix_attn_args;

int    gqa_prefix_attn_check(const gqa_prefix_attn_args * args);
size_t gqa_prefix_attn_workspace_size(const gqa_prefix_attn_args * args);
int    gqa_prefix_attn_launch(const gqa_prefix_attn_args * args, void * stream);

#ifdef __cplusplus
}
#endif
#endif /* GQA_BATCH_H */
