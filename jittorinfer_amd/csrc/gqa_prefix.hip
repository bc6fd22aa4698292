// Attention of one new token of every sequence where groups of sequences share their first rows (include/gqa_batch.h), for gfx950: three launches.
//
//   1. the groups' prefixes, a block of rows (member, head) against the shared keys, by the kernel of gqa_batch_kernel.hpp; every block is left as pieces (o, m, l)
//   2. the rows behind them, a sequence at a time, by gqa_attn's kernel; every head is left as pieces
//   3. the join, here: out = sum_i o_i 2^(m_i - M) / sum_i l_i 2^(m_i - M) over the pieces of both, in the order of the rows
//
// The keys of a prefix are read once a block of rows -- 128, 64 or 32 of them by the rows a group on average, groups of one among them -- where gqa_attn reads them once a sequence; a
// group's blocks find them in the caches.  (64 users, 4 / 16 / 32 of them behind 8192 shared rows, each of the others a group of one or in no group: 125 / 117 / 96 or 134 / 120 / 91 us; 16
// heads on 4 of 64 44 / 43 / 41 or 47 / 46 / 42, of 256 149 / 132 / 106 or 163 / 145 / 109.)  32 users behind 8192 shared rows (32 heads on 8 of 128): 46 us, of
// which the prefix is 25, the rows behind it 12.4 and the join 6.9 (8192 pieces' rows); 16 would be the bytes, and gqa_attn takes 142.  Each launch waits for lengths, page ids and
// rows in turn, and for the one before it.  Five users behind 100000 rows: 102 us (gqa_attn 289), 4.0 TB/s of the call.

#include <limits.h>

#include "gqa_attn.hpp"
#include "gqa_batch.hpp"

using namespace mla;
using namespace mla::gqa;

namespace {

// Grid: x = sequences, y = KV heads.  A thread takes 4 columns of a head at a time and, where a group's heads are few, one of several shares of the pieces: those of the
// prefix first, then those behind it; AHEAD of them are under way at a time.
constexpr int JOIN = 256, AHEAD = 4;
template <bool F16>
__global__ void __launch_bounds__(JOIN) gqa_prefix_join_kernel(const BatchP p, const AttnPieces a, const int bm, const int dv) {
    __shared__ f32x4  sh_o[JOIN];
    __shared__ float2 sh_ml[JOIN];
    const int b = blockIdx.x, kvh = blockIdx.y, G = p.group, n_el = G * (dv / 4);
    const int g = p.shared_group[b];
    const int n = min(min(max(a.seq_lens[b], 0), a.cap), a.mask_len);
    const bool has = g >= 0 && min(p.shared[b], p.mask_len) > 0, behind = n > a.behind[b];
    int64_t item0 = 0;
    int     row0 = 0;
    if (has) {
        const int q0 = min(max(p.q_starts[g], 0), p.n_tok);
        row0 = (b - q0) * G;
        item0 = (int64_t) q0 * G / bm + g;
    }
    // shares of the pieces: as many as there are threads for (a power of two)
    int shares = 1;
    while (shares * 2 * n_el <= JOIN) shares *= 2;
    for (int e0 = 0; e0 < n_el; e0 += JOIN) {
        const int e = shares > 1 ? (int) threadIdx.x % n_el : e0 + (int) threadIdx.x, share = shares > 1 ? (int) threadIdx.x / n_el : 0;
        const bool live = e < n_el && share < shares;
        const int r = live ? e % G : 0, c0 = live ? e / G * 4 : 0, h = kvh * G + r;
        float M = -INFINITY, L = 0.f;
        f32x4 o = { 0.f, 0.f, 0.f, 0.f };
        if (live) {
            // the prefix's pieces: runs v0 .. v0 + n0 - 1; those behind it: runs v1 .. v1 + n1 - 1, or one result
            const int row = row0 + r, j = row / bm, rr = row - j * bm;
            const int at = (((c0 >> 5) * 4 + ((c0 >> 3) & 3)) * (bm / 32) + (rr >> 5)) * 64 + ((c0 >> 2) & 1) * 32 + (rr & 31);
            int4 it = make_int4(0, 0, -1, 0);
            int2 i2 = make_int2(0, -1);
            const int hb = a.quad ? kvh >> 2 : kvh * a.row_blocks + r / a.rows, row2 = a.quad ? (kvh & 3) * G + r : r % a.rows;
            if (has) it = p.items[(item0 + j) * p.n_head_kv + kvh];
            if (behind) i2 = a.items[(int64_t) b * a.head_blocks + hb];
            const int v1 = i2.x >> 1, n0 = it.z - it.y + 1, n1 = i2.y - v1 + 1;
            for (int i0 = share; i0 < n0 + n1; i0 += shares * AHEAD) {
                float2 ml[AHEAD];
                f32x4  x[AHEAD];
#pragma unroll
                for (int k = 0; k < AHEAD; k++) {                     // (pieces past the last repeat it, without weight)
                    const int i = min(i0 + k * shares, n0 + n1 - 1);
                    const float2 * mls;
                    const float *  os;
                    if (i < n0) {
                        const int64_t slot = i ? 2 * (int64_t) (it.y + i) : it.x;
                        mls = p.part_ml + slot * bm + rr; os = p.part_o + slot * bm * dv + at * 4;
                    } else if (n1 == 1) {
                        mls = a.whole_ml + (int64_t) b * p.n_head + h; os = a.whole_o + ((int64_t) b * p.n_head + h) * dv + c0;
                    } else {
                        const int64_t slot = i > n0 ? 2 * (int64_t) (v1 + i - n0) : i2.x;
                        mls = a.part_ml + slot * a.rows + row2; os = a.part_o + (slot * a.rows + row2) * dv + c0;
                    }
                    ml[k] = *mls; x[k] = *(const f32x4 *) os;
                    if (i0 + k * shares >= n0 + n1) ml[k].y = 0.f;
                }
                float top = M;
#pragma unroll
                for (int k = 0; k < AHEAD; k++) if (ml[k].y != 0.f) top = fmaxf(top, ml[k].x);
                const float f = M == top ? 1.f : fast_exp2(M - top);
                o *= f; L *= f; M = top;
#pragma unroll
                for (int k = 0; k < AHEAD; k++) {
                    if (ml[k].y == 0.f) continue;                     // (an empty piece has no sums)
                    const float w = fast_exp2(ml[k].x - top);
                    o += x[k] * w; L += ml[k].y * w;
                }
            }
        }
        if (shares > 1) {
            sh_o[threadIdx.x] = o; sh_ml[threadIdx.x] = make_float2(M, L);
            __syncthreads();
            if (!live || share) return;
            for (int q = 1; q < shares; q++) {
                const float2 ml = sh_ml[q * n_el + e];
                if (ml.y == 0.f) continue;
                const float top = fmaxf(M, ml.x), f = M == top ? 1.f : fast_exp2(M - top), w = fast_exp2(ml.x - top);
                o = o * f + sh_o[q * n_el + e] * w; L = L * f + ml.y * w; M = top;
            }
        }
        if (!live) continue;
        o *= L == 0.f ? 0.f : 1.f / L;                                // (a NaN stays one)
        *(u32x2 *) (p.dst + (int64_t) b * p.d_nb2 + (int64_t) h * p.d_nb1 + c0 * 2) = u32x2{ pair16<F16>(o.x, o.y), pair16<F16>(o.z, o.w) };
    }
}

BatchCall call_of(const gqa_prefix_attn_args * a) {
    return BatchCall{ a->n_seq, a->n_prefix, a->n_head, a->n_head_kv, a->dk, a->dv, a->type, a->n_workgroups, a->scale, a->logit_softcap, a->q, a->q_nb1, a->q_nb2, a->prefix_starts, a->k, a->v,
                      a->bt_stride >= 0 && a->bt_stride < INT_MAX ? a->bt_stride * PAGE : INT64_MAX, a->mask, a->mask_nb1, a->mask_ne0, a->dst, a->d_nb1, a->d_nb2 };
}
// gqa_attn's call for what is behind the prefixes (or for all rows)
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
// The prefixes by themselves, or every sequence whole by gqa_attn: a table with room for less than 2^28 bytes of rows (the last cache's size) has the shared ones read from caches again
// and again, for less than the two further launches take.  us, prefixes by themselves / gqa_attn, 512 .. 8192 shared rows and 200 own ones a user, 32 heads on 8 of 128:
// 4 users with room for 13 MB 31 / 12, 38 MB 30 / 15, 138 MB 37 / 30; 16 of one group 50 MB 31 / 15, 151 MB 34 / 26, 285 MB 36 / 38, 554 MB 35 / 86; 64 of 8 groups 201 MB 40 / 31, 336 MB
// 41 / 47, 604 MB 42 / 93; 16 on 4 of 64: 138 MB 27 / 25, 285 MB 32 / 36, 554 MB 36 / 61; 16 on 4 of 256: 151 MB 42 / 28, 285 MB 44 / 46, 336 MB 45 / 34, 604 MB 49 / 52.
// So with as many groups as sequences, none of which has two then (or others have none): 64 users alone with 2000 rows each 109 / 100, 40 / 31 (16 on 4 of 64), 110 / 98 (of 256); one
// user's 100000 rows 122 / 87, 26 / 26, 104 / 82.
bool apart(const gqa_prefix_attn_args * a) {
    if (a->n_workgroups > 0) return a->n_prefix > 0;
    return a->n_prefix > 0 && a->n_prefix < a->n_seq && 2.0 * a->n_seq * a->bt_stride * PAGE * a->n_head_kv * (a->dk + a->dv) >= (double) (1 << 28);
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
    return !apart(a) ? gqa_attn_workspace_size(&t) : batch_plan(call_of(a), true).bytes + shared_bytes(a) + attn_behind_size(&t);
}
extern "C" int gqa_prefix_attn_launch(const gqa_prefix_attn_args * a, void * stream) {
    const int rc = gqa_prefix_attn_check(a);
    if (rc || a->n_seq == 0) return rc;
    if (!a->workspace || ((uintptr_t) a->workspace & 255) || a->workspace_size < gqa_prefix_attn_workspace_size(a)) return MLA_ERR_WORKSPACE;
    const gqa_attn_args t = attn_of(a);
    if (!apart(a)) return gqa_attn_launch(&t, stream);
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
