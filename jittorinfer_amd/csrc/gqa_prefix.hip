// Attention of one new token of every sequence where groups of sequences share their first rows (include/gqa_batch.h), for gfx950: three launches.
//
//   1. the groups' prefixes, a block of rows (member, head) against the shared keys, by the kernel of gqa_batch_kernel.hpp; every block is left as pieces (o, m, l)
//   2. the rows behind them, a sequence at a time, by gqa_attn's kernel; every head is left as pieces
//   3. the join, here: out = sum_i o_i 2^(m_i - M) / sum_i l_i 2^(m_i - M) over the pieces of both, in the order of the rows
//
// The keys of a prefix are read once a group and KV head for up to 128 rows, where gqa_attn reads them once a sequence.

#include <limits.h>

#include "gqa_attn.hpp"
#include "gqa_batch.hpp"

using namespace mla;
using namespace mla::gqa;

namespace {

// Grid: x = sequences, y = KV heads.  A thread takes 4 columns of a head at a time.
template <bool F16>
__global__ void __launch_bounds__(256) gqa_prefix_join_kernel(const BatchP p, const AttnPieces a, const int bm, const int dv) {
    const int b = blockIdx.x, kvh = blockIdx.y, G = p.group;
    // the prefix's pieces
    const int g = p.shared_group[b], shared = min(p.shared[b], p.mask_len);
    int4 it = make_int4(0, 0, 0, 0);
    int  pre = 0, pre_row = 0;
    if (g >= 0 && shared > 0) {
        const int q0 = min(max(p.q_starts[g], 0), p.n_tok), row = (b - q0) * G, j = row / bm;
        // (a sequence's heads may lie in two blocks: the others' pieces are looked up with them)
        it = p.items[((int64_t) q0 * G / bm + g + j) * p.n_head_kv + kvh];
        pre = it.z - it.y + 1; pre_row = row;
    }
    const int n = min(min(max(a.seq_lens[b], 0), a.cap), a.mask_len);
    const bool behind = n > a.behind[b];
    for (int e = threadIdx.x; e < G * (dv / 4); e += 256) {
        const int r = e % G, c0 = e / G * 4;
        float M = -INFINITY, L = 0.f;
        f32x4 o = { 0.f, 0.f, 0.f, 0.f };
        auto add = [&](float2 ml, const f32x4 * from) {               // pieces in order, relative to the largest reference so far
            if (ml.y == 0.f) return;                                  // (an empty piece has no sums)
            const f32x4 x = *from;
            const float top = fmaxf(M, ml.x), f = M == top ? 1.f : fast_exp2(M - top), w = fast_exp2(ml.x - top);
            o = o * f + x * w; L = L * f + ml.y * w; M = top;
        };
        if (pre) {
            const int row = pre_row + r, j = row / bm, rr = row - j * bm;
            int4 mine = it;
            if (j != pre_row / bm) {
                const int q0 = min(max(p.q_starts[g], 0), p.n_tok);
                mine = p.items[((int64_t) q0 * G / bm + g + j) * p.n_head_kv + kvh];
            }
            const int at = (((c0 >> 5) * 4 + ((c0 >> 3) & 3)) * (bm / 32) + (rr >> 5)) * 64 + ((c0 >> 2) & 1) * 32 + (rr & 31);
            for (int v = mine.y; v <= mine.z; v++) {
                const int64_t slot = v == mine.y ? mine.x : 2 * (int64_t) v;
                add(p.part_ml[slot * bm + rr], (const f32x4 *) p.part_o + slot * (bm * dv / 4) + at);
            }
        }
        if (behind) {
            const int h = kvh * G + r, hb = a.quad ? kvh >> 2 : kvh * a.row_blocks + r / a.rows, row = a.quad ? (kvh & 3) * G + r : r % a.rows;
            const int2 i2 = a.items[(int64_t) b * a.head_blocks + hb];
            const int  v0 = i2.x >> 1;
            if (v0 == i2.y) add(a.whole_ml[(int64_t) b * p.n_head + h], (const f32x4 *) (a.whole_o + ((int64_t) b * p.n_head + h) * dv + c0));
            else
                for (int v = v0; v <= i2.y; v++) {
                    const int64_t slot = v == v0 ? i2.x : 2 * (int64_t) v;
                    add(a.part_ml[slot * a.rows + row], (const f32x4 *) (a.part_o + (slot * a.rows + row) * dv + c0));
                }
        }
        o *= L == 0.f ? 0.f : 1.f / L;                                // (a NaN stays one)
        *(u32x2 *) (p.dst + (int64_t) b * p.d_nb2 + (int64_t) (kvh * G + r) * p.d_nb1 + c0 * 2) = u32x2{ pair16<F16>(o.x, o.y), pair16<F16>(o.z, o.w) };
    }
}

BatchCall call_of(const gqa_prefix_attn_args * a) {
    return BatchCall{ a->n_seq, a->n_prefix, a->n_head, a->n_head_kv, a->dk, a->dv, a->type, a->n_workgroups, a->scale, a->logit_softcap, a->q, a->q_nb1, a->q_nb2, a->prefix_starts, a->k, a->v,
                      a->bt_stride >= 0 && a->bt_stride < INT_MAX ? a->bt_stride * PAGE : INT64_MAX, a->mask, a->mask_nb1, a->mask_ne0, a->dst, a->d_nb1, a->d_nb2 };
}
// gqa_attn's call for what is behind the prefixes (or, without any, for all rows)
gqa_attn_args attn_of(const gqa_prefix_attn_args * a) {
    gqa_attn_args t = {};
    t.n_seq = a->n_seq; t.n_head = a->n_head; t.n_head_kv = a->n_head_kv; t.dk = a->dk; t.dv = a->dv; t.q_type = t.kv_type = t.dst_type = a->type;
    t.scale = a->scale; t.logit_softcap = a->logit_softcap; t.n_workgroups = a->n_workgroups;
    t.q = a->q; t.q_nb1 = a->q_nb1; t.q_nb2 = a->q_nb2; t.k = a->k; t.v = a->v; t.n_pages = a->n_pages;
    t.block_table = a->block_table; t.bt_stride = a->bt_stride; t.seq_lens = a->seq_lens;
    t.mask = a->mask; t.mask_nb1 = a->mask_nb1; t.mask_ne0 = a->mask_ne0;
    t.dst = a->dst; t.d_nb1 = a->d_nb1; t.d_nb2 = a->d_nb2; t.workspace = a->workspace; t.workspace_size = a->workspace_size;
    return t;
}
size_t shared_bytes(const gqa_prefix_attn_args * a) { return (2 * (size_t) a->n_seq * 4 + 255) & ~(size_t) 255; }

}  // namespace

extern "C" int gqa_prefix_attn_check(const gqa_prefix_attn_args * a) {
    if (!a) return MLA_ERR_NULL;
    if (a->n_prefix < 0) return MLA_ERR_BAD_SHAPE;
    if (a->n_seq > 0 && a->n_prefix > 0) {
        if (!a->prefix_starts || !a->prefix_lens) return MLA_ERR_NULL;
        if (a->dst == (const void *) a->prefix_lens) return MLA_ERR_UNSUPPORTED;
    }
    const gqa_attn_args t = attn_of(a);
    const int rc = gqa_attn_check(&t);
    return rc ? rc : batch_check(call_of(a));
}
extern "C" size_t gqa_prefix_attn_workspace_size(const gqa_prefix_attn_args * a) {
    if (gqa_prefix_attn_check(a) || a->n_seq == 0) return 0;
    const gqa_attn_args t = attn_of(a);
    return a->n_prefix == 0 ? gqa_attn_workspace_size(&t) : batch_plan(call_of(a), true).bytes + shared_bytes(a) + attn_behind_size(&t);
}
extern "C" int gqa_prefix_attn_launch(const gqa_prefix_attn_args * a, void * stream) {
    const int rc = gqa_prefix_attn_check(a);
    if (rc || a->n_seq == 0) return rc;
    if (!a->workspace || ((uintptr_t) a->workspace & 255) || a->workspace_size < gqa_prefix_attn_workspace_size(a)) return MLA_ERR_WORKSPACE;
    const gqa_attn_args t = attn_of(a);
    if (a->n_prefix == 0) return gqa_attn_launch(&t, stream);
    const BatchCall   c  = call_of(a);
    const BatchPlan   pl = batch_plan(c, true);
    const hipStream_t st = (hipStream_t) stream;
    char * ws = (char *) a->workspace;
    BatchP p;
    batch_fill(p, c, pl, ws);
    ws += pl.bytes;
    p.block_table = a->block_table; p.bt_stride = a->bt_stride; p.n_pages = a->n_pages; p.lens = a->prefix_lens; p.own_lens = a->seq_lens;
    p.shared = (int32_t *) ws; p.shared_group = p.shared + a->n_seq;
    ws += shared_bytes(a);
    const bool f16 = a->type == MLA_TYPE_F16;
    hipError_t e = f16 ? batch_launch<true>(p, pl, a->dk, st) : batch_launch<false>(p, pl, a->dk, st);
    if (e != hipSuccess) return (int) e;
    AttnPieces pieces;
    if ((e = attn_behind(&t, p.shared, ws, pieces, st)) != hipSuccess) return (int) e;
    const dim3 grid((unsigned) a->n_seq, (unsigned) a->n_head_kv);
    if (f16) hipLaunchKernelGGL(gqa_prefix_join_kernel<true>, grid, dim3(256), 0, st, p, pieces, pl.bm, a->dv);
    else     hipLaunchKernelGGL(gqa_prefix_join_kernel<false>, grid, dim3(256), 0, st, p, pieces, pl.bm, a->dv);
    return (int) hipGetLastError();
}
