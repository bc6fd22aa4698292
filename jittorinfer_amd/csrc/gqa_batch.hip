// Entry points of attention of many query rows over the same keys (include/gqa_batch.h): argument checks and plans; the kernels are in gqa_batch_kernel.hpp.

#include <float.h>
#include <limits.h>
#include <math.h>

#include "gqa_batch.hpp"

using namespace mla;
using namespace mla::gqa;

namespace {

template <typename A> BatchCall call_of(const A * a, int64_t cap) {
    return BatchCall{ a->n_tok, a->n_seq, a->n_head, a->n_head_kv, a->dk, a->dv, a->type, a->n_workgroups, a->scale, a->logit_softcap, a->q, a->q_nb1, a->q_nb2, a->q_starts, a->k, a->v, cap,
                 a->mask, a->mask_nb1, a->mask_ne0, a->dst, a->d_nb1, a->d_nb2 };
}

}  // namespace

BatchPlan mla::gqa::batch_plan(const BatchCall & c, bool whole_blocks) {
    BatchPlan pl;
    const int     group = c.n_head / c.n_head_kv;
    const int64_t rows = ((int64_t) c.n_tok * group + c.n_seq - 1) / c.n_seq;     // of a sequence, on average
    // Waves along the keys where rows are few; and up to 192 of them where there are few runs of keys (KV heads of all groups), which then lie in more workgroups'
    // hands and are read again from the caches.  Four along the keys / two and two / four along the rows, us, 4000 rows of keys, 32 heads on 8 of 128: 1 x 8
    // tokens (32 rows) 24 / 30 / 35, 1 x 16 (64) 23 / 31 / 36, 1 x 48 (192) 32 / 36 / 41, 16 x 8 55 / 62 / 73, 16 x 16 68 / 64 / 75, 16 x 24 (96) 124 / 73 / 77, 16 x 48 232 /
    // 147 / 100; 16 on 4 of 64: 16 x 16 28 / 32 / 46, 16 x 32 35 / 33 / 46; 16 on 4 of 256 (two and two, four along the rows): 1 x 32 49 / 59, 16 x 16 67 / 91, 16 x 32 99 / 93.
    const int64_t runs = (int64_t) c.n_seq * c.n_head_kv;
    if (rows <= 64 || (rows <= 192 && runs <= 32)) pl.shape = c.dk <= 128 ? FOUR_KEYS : TWO_TWO;
    else pl.shape = rows <= 128 && c.dk <= 128 ? TWO_TWO : FOUR_ROWS;
    pl.bm     = pl.shape == FOUR_KEYS ? 32 : pl.shape == TWO_TWO ? 64 : 128;
    const int64_t blocks = (int64_t) c.n_tok * group / pl.bm + c.n_seq;
    pl.blocks = blocks < INT_MAX ? (int) blocks : INT_MAX;
    const int64_t tiles = (c.cap + 63) / 64 < INT_MAX ? (c.cap + 63) / 64 : INT_MAX, fill = 256 * batch_wg_per_cu(c.dk, pl.shape, !c.mask && c.logit_softcap == 0.f);
    const int64_t most = c.n_workgroups > 0 ? c.n_workgroups : fill, have = tiles > most ? most : tiles * pl.blocks > most ? most : tiles * pl.blocks * c.n_head_kv;
    pl.n_wg = (int) (have < 1 ? 1 : have < most ? have : most);
    size_t at = 0;
    auto take = [&](size_t n) { const size_t o = at; at += (n + 255) & ~(size_t) 255; return o; };
    const size_t slots = 2 * (size_t) pl.n_wg + (whole_blocks ? (size_t) pl.blocks * c.n_head_kv : 0);
    take(slots * pl.bm * c.dv * 4);
    pl.off_ml    = take(slots * pl.bm * 8);
    pl.off_items = take((size_t) pl.blocks * c.n_head_kv * 16);
    pl.off_tasks = take((size_t) pl.n_wg * 16);
    // (four blocks a workgroup of one sequence are taken whole in any case: no more than an eighth of the time is lost at the end)
    const int64_t full = (int64_t) c.n_tok * group / pl.bm * c.n_head_kv;
    pl.deal = whole_blocks || c.n_workgroups > 0 ? RUNS : c.n_seq == 1 && full >= 4 * fill ? WHOLE : EITHER;
    pl.bytes = at;
    return pl;
}

namespace {
int check_pool(const gqa_pool & c) {
    if (!c.data) return MLA_ERR_NULL;
    if (!al16(c.data) || (c.nb_page & 15) || (c.nb_row & 15) || (c.nb_head & 15)) return MLA_ERR_BAD_ALIGNMENT;
    return c.nb_page < 0 || c.nb_head < 0 || c.nb_row < 0 || c.nb_row > (1 << 23) ? MLA_ERR_BAD_SHAPE : 0;   // (a tile's rows lie within 32 bits)
}

}  // namespace

int mla::gqa::batch_check(const BatchCall & c) {
    if (c.type != MLA_TYPE_BF16 && c.type != MLA_TYPE_F16) return MLA_ERR_BAD_TYPE;
    if (c.n_tok < 0 || c.n_seq < 0 || c.n_head < 1 || c.n_head_kv < 1 || c.n_head % c.n_head_kv || c.n_workgroups < 0 || c.n_workgroups > 65536) return MLA_ERR_BAD_SHAPE;
    if (c.dk == 64 || c.dk == 128 || c.dk == 256 ? c.dv != c.dk : c.dk != 192 || c.dv != 128) return MLA_ERR_UNSUPPORTED;
    if (!(c.logit_softcap >= 0.f && c.logit_softcap <= FLT_MAX)) return MLA_ERR_UNSUPPORTED;
    if (c.n_tok == 0 || c.n_seq == 0) return 0;
    if (!c.q || !c.dst) return MLA_ERR_NULL;
    if (!c.q_starts && c.n_tok % c.n_seq) return MLA_ERR_BAD_SHAPE;
    if (c.cap >= (int64_t) 1 << 30 || (int64_t) c.n_tok * c.n_head >= (int64_t) 1 << 31 || c.n_head_kv > 65535) return MLA_ERR_BAD_SHAPE;
    int rc = c.cap ? check_pool(c.k) : 0;                          // (states of no row need not lie anywhere)
    if (!rc && c.cap) rc = check_pool(c.v);
    if (rc) return rc;
    if (!al16(c.q) || (c.q_nb1 & 15) || (c.q_nb2 & 15) || ((uintptr_t) c.dst & 7) || (c.d_nb1 & 7) || (c.d_nb2 & 7)) return MLA_ERR_BAD_ALIGNMENT;
    if (c.mask) {
        if (((uintptr_t) c.mask & 1) || (c.mask_nb1 & 1)) return MLA_ERR_BAD_ALIGNMENT;
        if (c.mask_ne0 < 0) return MLA_ERR_BAD_SHAPE;
    }
    // what is written is nothing that is read (by its address alone: strides may lay one between the other's rows)
    if (c.dst == c.q || c.dst == c.k.data || c.dst == c.v.data || c.dst == c.mask || c.dst == (const void *) c.q_starts) return MLA_ERR_UNSUPPORTED;
    const BatchPlan pl = batch_plan(c, false);
    // (a launch holds fewer than 2^32 threads, and items are counted in 31 bits)
    return (uint64_t) pl.blocks * c.n_head_kv >= (1 << 24) ? MLA_ERR_BAD_SHAPE : 0;
}

void mla::gqa::batch_fill(BatchP & p, const BatchCall & c, const BatchPlan & pl, char * ws) {
    p.q = (const char *) c.q; p.q_nb1 = c.q_nb1; p.q_nb2 = c.q_nb2;
    p.k = (const char *) c.k.data; p.k_page = c.k.nb_page; p.k_head = c.k.nb_head; p.k_row = (int) c.k.nb_row;
    p.v = (const char *) c.v.data; p.v_page = c.v.nb_page; p.v_head = c.v.nb_head; p.v_row = (int) c.v.nb_row;
    p.block_table = nullptr; p.bt_stride = p.n_pages = 0; p.kv_starts = p.lens = p.own_lens = nullptr; p.shared = p.shared_group = nullptr;
    p.q_starts = c.q_starts; p.per = c.n_tok / c.n_seq;
    p.mask = (const char *) c.mask; p.mask_nb1 = c.mask_nb1; p.mask_len = c.mask && c.mask_ne0 < c.cap ? (int) c.mask_ne0 : (int) c.cap;
    p.dst = (char *) c.dst; p.d_nb1 = c.d_nb1; p.d_nb2 = c.d_nb2;
    p.scale_log2 = fabsf(c.scale) * LOG2E; p.mask_unit = 1.f / fabsf(c.scale); p.flip = c.scale < 0.f ? 0x80008000u : 0u;
    // (a cap so small or large that these leave f32: the largest number does the same)
    p.cap_in  = c.logit_softcap > 0.f ? fminf(fabsf(c.scale) / c.logit_softcap, FLT_MAX) : 0.f;
    p.cap_out = fminf(c.logit_softcap * LOG2E, FLT_MAX);
    p.causal = 0; p.window = 0; p.n_grp = c.n_seq; p.n_tok = c.n_tok; p.n_head = c.n_head; p.n_head_kv = c.n_head_kv; p.group = c.n_head / c.n_head_kv; p.per_head = 1.0 / p.group;
    p.cap = (int) c.cap; p.n_wg = pl.n_wg;
    // A piece of a block is bm x dv numbers to write and to read again: 4 tiles or more a workgroup.  1, 2, 4, 8, 16 of them, us: 8 tokens behind 4000 rows 24.0, 24.3, 23.2, 28.3,
    // 38.0; 64 tokens 79, 79, 41, 39, 45; 32 users behind 8192 shared rows 49.6, 49.2, 47.5, 46.3, 54.3; one token of 16 over 1500 states 29.6, 29.4, 29.4, 30.7, 34.4.
    p.min_tiles = c.n_workgroups > 0 ? 1 : 4;
    p.part_o = (float *) ws; p.part_ml = (float2 *) (ws + pl.off_ml); p.items = (int4 *) (ws + pl.off_items);
    p.tasks = (int4 *) (ws + pl.off_tasks); p.blocks = pl.blocks; p.deal = pl.deal;
}

namespace {
template <typename A> int ready(const A * a, const BatchPlan & pl) {
    return !a->workspace || ((uintptr_t) a->workspace & 255) || a->workspace_size < pl.bytes ? MLA_ERR_WORKSPACE : 0;
}
int launch(const BatchP & p, const BatchCall & c, const BatchPlan & pl, void * stream) {
    return (int) (c.type == MLA_TYPE_F16 ? batch_launch<true>(p, pl, c.dk, (hipStream_t) stream) : batch_launch<false>(p, pl, c.dk, (hipStream_t) stream));
}

}  // namespace

// ---------------------------------------------------------------- prompts

static BatchCall prompt_call(const gqa_prompt_attn_args * a) { return call_of(a, a->bt_stride >= 0 && a->bt_stride < INT_MAX ? a->bt_stride * PAGE : INT64_MAX); }

extern "C" int gqa_prompt_attn_check(const gqa_prompt_attn_args * a) {
    if (!a) return MLA_ERR_NULL;
    if (a->window < 0) return MLA_ERR_BAD_SHAPE;
    if (a->n_tok > 0 && a->n_seq > 0) {
        if (!a->block_table || !a->seq_lens) return MLA_ERR_NULL;
        if (a->n_pages < 1 || a->bt_stride < 1) return MLA_ERR_BAD_SHAPE;
        if (a->dst && (a->dst == (const void *) a->block_table || a->dst == (const void *) a->seq_lens)) return MLA_ERR_UNSUPPORTED;
    }
    return batch_check(prompt_call(a));
}
extern "C" size_t gqa_prompt_attn_workspace_size(const gqa_prompt_attn_args * a) {
    return gqa_prompt_attn_check(a) || a->n_tok == 0 || a->n_seq == 0 ? 0 : batch_plan(prompt_call(a), false).bytes;
}
extern "C" int gqa_prompt_attn_launch(const gqa_prompt_attn_args * a, void * stream) {
    int rc = gqa_prompt_attn_check(a);
    if (rc || a->n_tok == 0 || a->n_seq == 0) return rc;
    const BatchCall      c  = prompt_call(a);
    const BatchPlan pl = batch_plan(c, false);
    if ((rc = ready(a, pl))) return rc;
    BatchP p;
    batch_fill(p, c, pl, (char *) a->workspace);
    p.block_table = a->block_table; p.bt_stride = a->bt_stride; p.n_pages = a->n_pages; p.lens = a->seq_lens;
    p.causal = a->causal != 0; p.window = a->window;
    return launch(p, c, pl, stream);
}

// ---------------------------------------------------------------- an encoder's states

static BatchCall cross_call(const gqa_cross_attn_args * a) { return call_of(a, a->n_kv); }

extern "C" int gqa_cross_attn_check(const gqa_cross_attn_args * a) {
    if (!a) return MLA_ERR_NULL;
    if (a->n_kv < 0) return MLA_ERR_BAD_SHAPE;
    if (a->n_tok > 0 && a->n_seq > 0) {
        if (a->kv_starts && (a->k.nb_page || a->v.nb_page)) return MLA_ERR_BAD_SHAPE;
        if (a->dst && (a->dst == (const void *) a->kv_starts || a->dst == (const void *) a->kv_lens)) return MLA_ERR_UNSUPPORTED;
    }
    return batch_check(cross_call(a));
}
extern "C" size_t gqa_cross_attn_workspace_size(const gqa_cross_attn_args * a) {
    return gqa_cross_attn_check(a) || a->n_tok == 0 || a->n_seq == 0 ? 0 : batch_plan(cross_call(a), false).bytes;
}
extern "C" int gqa_cross_attn_launch(const gqa_cross_attn_args * a, void * stream) {
    int rc = gqa_cross_attn_check(a);
    if (rc || a->n_tok == 0 || a->n_seq == 0) return rc;
    const BatchCall      c  = cross_call(a);
    const BatchPlan pl = batch_plan(c, false);
    if ((rc = ready(a, pl))) return rc;
    BatchP p;
    batch_fill(p, c, pl, (char *) a->workspace);
    p.kv_starts = a->kv_starts; p.lens = a->kv_lens;
    return launch(p, c, pl, stream);
}
