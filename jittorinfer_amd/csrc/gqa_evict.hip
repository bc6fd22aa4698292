// Eviction from a paged cache by accumulated attention weight (include/gqa_attn.h), for gfx950: which rows stay, and their way up.
//
// Selection (gqa_select_kernel, a workgroup per (sequence, KV head)): the weights' bits, made monotone, are searched digit by digit for the
// smallest weight that stays (11 + 11 + 10 bits, a histogram in LDS each), then one pass in the order of the rows writes the rows that stay:
// those above it, and of those equal to it the first ones, counted by a scan.  Reads the weights four times, from HBM once.
//
// Moving (gqa_move_kernel): row kept[j] goes to row j <= kept[j], in place and without scratch, read once and written once.  A workgroup takes a
// stripe of a few 16-byte columns of one (sequence, KV head) and all its rows, in chunks from the front: the chunk's sources into registers, a
// barrier, then the stores.  What a chunk overwrites (rows below its end) no later chunk reads (sources lie at or behind their targets), and
// no other workgroup touches these columns.

#include "mla_common.hpp"
#include "../../include/gqa_attn.h"

using namespace mla;

namespace {

constexpr int PAGE = MLA_PAGE_TOKENS;
constexpr int SEL_THREADS = 1024, SEL_PER = 8;       // rows a thread takes at a time, consecutive
constexpr int BINS = 2048;

struct EvictP {
    const char * w; int64_t w_nb1, w_nb2;
    char * wd; int64_t wd_nb1, wd_nb2;
    int32_t * kept, * new_lens;
    const int32_t * seq_lens, * block_table;
    int64_t bt_stride, n_pages, cap;
    int n_seq, n_head_kv, n_keep, n_sink, n_recent;
    char * k; int64_t k_page, k_row, k_head;
    char * v; int64_t v_page, v_row, v_head;
    int k_units, v_units, k_stripes;                  // units of 16 (or 4) bytes of a head's row; stripes of the keys come first
};

__device__ __forceinline__ int len_of(const EvictP & p, int b) {
    const int64_t n = p.seq_lens[b];
    return (int) (n < 0 ? 0 : n > p.cap ? p.cap : n);
}

// Monotone: a < b as numbers <=> key(a) < key(b); -0 as +0, NaN below everything.
__device__ __forceinline__ unsigned key_of(float x) {
    if (x != x) return 0u;
    const unsigned u = __float_as_uint(x + 0.0f);
    return (u & 0x80000000u) ? ~u : u | 0x80000000u;
}

__device__ __forceinline__ int scan_wave(int v, int lane) {       // inclusive
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) { const int o = __shfl_up(v, d, 64); if (lane >= d) v += o; }
    return v;
}

__global__ void __launch_bounds__(SEL_THREADS) gqa_select_kernel(const EvictP p) {
    __shared__ unsigned hist[BINS];
    __shared__ int      part[16];
    __shared__ unsigned sh_digit;
    __shared__ int      sh_left;
    const int b = blockIdx.x / p.n_head_kv, h = blockIdx.x - b * p.n_head_kv;
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const int n = len_of(p, b), m = min(n, p.n_keep);
    const float * w  = (const float *) (p.w + (int64_t) b * p.w_nb2 + (int64_t) h * p.w_nb1);
    float *       wd = (float *) (p.wd + (int64_t) b * p.wd_nb2 + (int64_t) h * p.wd_nb1);
    int32_t *     kept = p.kept + (int64_t) blockIdx.x * p.n_keep;
    if (h == 0 && tid == 0) p.new_lens[b] = m;
    if (n <= p.n_keep) {                                           // nothing leaves
        for (int i = tid; i < p.n_keep; i += SEL_THREADS) kept[i] = i < n ? i : -1;
        for (int64_t i = tid; i < p.cap; i += SEL_THREADS) wd[i] = i < n ? w[i] : 0.f;
        return;
    }
    const int  c0 = p.n_sink, c1 = n - p.n_recent;                 // the rows that compete (c0 < c1: n_sink + n_recent <= n_keep < n)
    const int  places = p.n_keep - p.n_sink - p.n_recent;
    const bool vec = ((uintptr_t) w & 15) == 0;
    auto load8 = [&](int i0, float (&x)[SEL_PER]) {                // rows i0 .. i0 + 7; past the length: nothing is read
        if (vec && i0 + SEL_PER <= n) {
            const f32x4 a = *(const f32x4 *) (w + i0), c = *(const f32x4 *) (w + i0 + 4);
#pragma unroll
            for (int e = 0; e < 4; e++) { x[e] = a[e]; x[4 + e] = c[e]; }
        } else {
#pragma unroll
            for (int e = 0; e < SEL_PER; e++) x[e] = i0 + e < n ? w[i0 + e] : 0.f;
        }
    };

    unsigned prefix = 0;                                           // the digits found so far
    int      left = places;                                        // rows still to be taken among those that share them
    if (places > 0) {
        for (int pass = 0; pass < 3; pass++) {
            const int shift = pass == 0 ? 21 : pass == 1 ? 10 : 0, bits = pass == 2 ? 10 : 11;
            for (int i = tid; i < BINS; i += SEL_THREADS) hist[i] = 0;
            __syncthreads();
            for (int i0 = tid * SEL_PER; i0 < c1; i0 += SEL_THREADS * SEL_PER) {
                float x[SEL_PER];
                load8(i0, x);
#pragma unroll
                for (int e = 0; e < SEL_PER; e++) {
                    const int i = i0 + e;
                    const unsigned k = key_of(x[e]);
                    if (i >= c0 && i < c1 && (pass == 0 || (k >> (shift + bits)) == prefix)) atomicAdd(&hist[(k >> shift) & ((1u << bits) - 1)], 1u);
                }
            }
            __syncthreads();
            // the digit at which the rows from the top on reach `left`: thread t holds bins 2047 - 2t and 2046 - 2t
            const int hi = (int) hist[BINS - 1 - 2 * tid], lo = (int) hist[BINS - 2 - 2 * tid];
            int incl = scan_wave(hi + lo, lane);
            if (lane == 63) part[wave] = incl;
            __syncthreads();
            for (int q = 0; q < wave; q++) incl += part[q];
            const int above = incl - hi - lo;
            if (above < left && incl >= left) {
                const bool first = above + hi >= left;
                sh_digit = (unsigned) (BINS - 1 - 2 * tid - (first ? 0 : 1));
                sh_left  = left - above - (first ? 0 : hi);
            }
            __syncthreads();
            prefix = (prefix << bits) | sh_digit;
            left   = sh_left;
            __syncthreads();
        }
    }
    // prefix: the key of the smallest weight that stays, `left` rows of which do
    int taken = 0, ties = 0;                                       // rows before this chunk: surely kept, and equal to the smallest
    for (int base = 0; base < n; base += SEL_THREADS * SEL_PER) {
        const int i0 = base + tid * SEL_PER;
        float x[SEL_PER];
        load8(min(i0, n), x);
        int sure = 0, tie = 0;                                     // bit e: row i0 + e
#pragma unroll
        for (int e = 0; e < SEL_PER; e++) {
            const int i = i0 + e;
            if (i >= n) continue;
            const unsigned k = key_of(x[e]);
            if (i < c0 || i >= c1 || (places > 0 && k > prefix)) sure |= 1 << e;
            else if (places > 0 && k == prefix) tie |= 1 << e;
        }
        const int mine = __popc(sure) | (__popc(tie) << 16);      // (at most 8192 of either in a chunk)
        int incl = scan_wave(mine, lane);
        if (lane == 63) part[wave] = incl;
        __syncthreads();                                           // (also: every row of the chunk has been read before one is overwritten)
        int before = 0, all = 0;
        for (int q = 0; q < 16; q++) { if (q < wave) before += part[q]; all += part[q]; }
        before += incl - mine;
        int s = taken + (before & 0xffff), t = ties + (before >> 16);
#pragma unroll
        for (int e = 0; e < SEL_PER; e++) {
            const bool is_sure = sure >> e & 1, is_tie = tie >> e & 1;
            if (is_sure || (is_tie && t < left)) {
                const int j = s + min(t, left);
                kept[j] = i0 + e;
                wd[j]   = x[e];
            }
            s += is_sure; t += is_tie;
        }
        taken += all & 0xffff; ties += all >> 16;
        __syncthreads();
    }
    for (int64_t i = p.n_keep + tid; i < p.cap; i += SEL_THREADS) wd[i] = 0.f;
}

constexpr int MOVE_THREADS = 1024, MOVE_SU = 4, MOVE_R = 8;        // units a row of a stripe, rows a thread has in flight

template <typename T>
__global__ void __launch_bounds__(MOVE_THREADS) gqa_move_kernel(const EvictP p) {
    const int b = blockIdx.y / p.n_head_kv, h = blockIdx.y - b * p.n_head_kv;
    if (len_of(p, b) <= p.n_keep) return;
    const bool is_k = (int) blockIdx.x < p.k_stripes;
    const int  unit = (is_k ? (int) blockIdx.x : (int) blockIdx.x - p.k_stripes) * MOVE_SU + (int) threadIdx.x % MOVE_SU;
    const bool has = unit < (is_k ? p.k_units : p.v_units);
    char *     base = (is_k ? p.k + h * p.k_head : p.v + h * p.v_head) + (int64_t) unit * sizeof(T);
    const int64_t nb_page = is_k ? p.k_page : p.v_page, nb_row = is_k ? p.k_row : p.v_row;
    const int32_t * kept = p.kept + (int64_t) blockIdx.y * p.n_keep;
    const int32_t * bt = p.block_table + (int64_t) b * p.bt_stride;
    constexpr int STEP = MOVE_THREADS / MOVE_SU;
    for (int j0 = (int) threadIdx.x / MOVE_SU; j0 - (int) threadIdx.x / MOVE_SU < p.n_keep; j0 += STEP * MOVE_R) {
        T      x[MOVE_R];
        char * to[MOVE_R];
#pragma unroll
        for (int r = 0; r < MOVE_R; r++) {
            const int j = j0 + r * STEP;
            to[r] = nullptr;
            if (has && j < p.n_keep) {
                const int src = kept[j];
                if (src != j) {
                    const int64_t from = bt[src / PAGE], into = bt[j / PAGE];
                    if (from >= 0 && from < p.n_pages && into >= 0 && into < p.n_pages) {
                        x[r]  = *(const T *) (base + from * nb_page + (src % PAGE) * nb_row);
                        to[r] = base + into * nb_page + (j % PAGE) * nb_row;
                    }
                }
            }
        }
        asm volatile("s_waitcnt vmcnt(0)" ::: "memory");           // the chunk's sources are here before anyone overwrites one
        __syncthreads();
#pragma unroll
        for (int r = 0; r < MOVE_R; r++) if (to[r]) *(T *) to[r] = x[r];
    }
}

int check_pool(const gqa_pool & c, int row_bytes) {
    if (!c.data) return MLA_ERR_NULL;
    if (((uintptr_t) c.data & 3) || (c.nb_page & 3) || (c.nb_row & 3) || (c.nb_head & 3) || (row_bytes & 3)) return MLA_ERR_BAD_ALIGNMENT;
    return c.nb_page < 0 || c.nb_row < 0 || c.nb_head < 0 || row_bytes < 4 || row_bytes > (1 << 20) ? MLA_ERR_BAD_SHAPE : 0;
}
bool wide(const gqa_pool & c, int row_bytes) { return !(((uintptr_t) c.data & 15) || (c.nb_page & 15) || (c.nb_row & 15) || (c.nb_head & 15) || (row_bytes & 15)); }

}  // namespace

extern "C" int gqa_evict_check(const gqa_evict_args * a) {
    if (!a) return MLA_ERR_NULL;
    if (a->n_seq < 0 || a->n_head_kv < 1 || a->n_keep < 1 || a->n_sink < 0 || a->n_recent < 0 || (int64_t) a->n_sink + a->n_recent > a->n_keep) return MLA_ERR_BAD_SHAPE;
    if (a->n_seq == 0) return 0;
    if (!a->weights || !a->weights_dst || !a->kept || !a->new_lens || !a->block_table || !a->seq_lens) return MLA_ERR_NULL;
    if (a->n_pages < 1 || a->bt_stride < 1 || a->bt_stride * PAGE >= ((int64_t) 1 << 30) || (int64_t) a->n_seq * a->n_head_kv > 65535) return MLA_ERR_BAD_SHAPE;
    int rc = check_pool(a->k, a->k_row_bytes);
    if (!rc && a->v.data) rc = check_pool(a->v, a->v_row_bytes);
    if (rc) return rc;
    if (((uintptr_t) a->weights & 3) || (a->w_nb1 & 3) || (a->w_nb2 & 3) || ((uintptr_t) a->weights_dst & 3) || (a->wd_nb1 & 3) || (a->wd_nb2 & 3)) return MLA_ERR_BAD_ALIGNMENT;
    if (a->weights == a->weights_dst && (a->w_nb1 != a->wd_nb1 || a->w_nb2 != a->wd_nb2)) return MLA_ERR_BAD_SHAPE;
    if (a->new_lens == a->seq_lens) return MLA_ERR_UNSUPPORTED;
    return 0;
}

extern "C" int gqa_evict_launch(const gqa_evict_args * a, void * stream) {
    const int rc = gqa_evict_check(a);
    if (rc) return rc;
    if (a->n_seq == 0) return 0;
    EvictP p;
    p.w = (const char *) a->weights; p.w_nb1 = a->w_nb1; p.w_nb2 = a->w_nb2;
    p.wd = (char *) a->weights_dst; p.wd_nb1 = a->wd_nb1; p.wd_nb2 = a->wd_nb2;
    p.kept = a->kept; p.new_lens = a->new_lens; p.seq_lens = a->seq_lens; p.block_table = a->block_table;
    p.bt_stride = a->bt_stride; p.n_pages = a->n_pages; p.cap = a->bt_stride * PAGE;
    p.n_seq = a->n_seq; p.n_head_kv = a->n_head_kv; p.n_keep = a->n_keep; p.n_sink = a->n_sink; p.n_recent = a->n_recent;
    p.k = (char *) a->k.data; p.k_page = a->k.nb_page; p.k_row = a->k.nb_row; p.k_head = a->k.nb_head;
    p.v = (char *) a->v.data; p.v_page = a->v.nb_page; p.v_row = a->v.nb_row; p.v_head = a->v.nb_head;
    const bool w16 = wide(a->k, a->k_row_bytes) && (!a->v.data || wide(a->v, a->v_row_bytes));
    const int  unit = w16 ? 16 : 4;
    p.k_units = a->k_row_bytes / unit; p.v_units = a->v.data ? a->v_row_bytes / unit : 0;
    p.k_stripes = (p.k_units + MOVE_SU - 1) / MOVE_SU;
    const unsigned stripes = (unsigned) (p.k_stripes + (p.v_units + MOVE_SU - 1) / MOVE_SU), groups = (unsigned) (a->n_seq * a->n_head_kv);
    hipLaunchKernelGGL(gqa_select_kernel, dim3(groups), dim3(SEL_THREADS), 0, (hipStream_t) stream, p);
    hipError_t e = hipGetLastError();
    if (e != hipSuccess) return (int) e;
    // (the rows' room is what the block table can hold: a table no wider than n_keep holds nothing to evict)
    if (p.cap <= a->n_keep) return 0;
    if (w16) hipLaunchKernelGGL(gqa_move_kernel<u32x4>, dim3(stripes, groups), dim3(MOVE_THREADS), 0, (hipStream_t) stream, p);
    else     hipLaunchKernelGGL(gqa_move_kernel<unsigned>, dim3(stripes, groups), dim3(MOVE_THREADS), 0, (hipStream_t) stream, p);
    return (int) hipGetLastError();
}
