// Eviction from a paged cache by accumulated attention weight (include/gqa_attn.h), for gfx950: which rows stay, and their way up.
//
// Selection (gqa_select_kernel, a workgroup per (sequence, KV head)): the weights' bits, made monotone, are searched digit by digit for the
// smallest weight that stays (11 + 11 + 10 bits, a histogram in LDS each), then one pass in the order of the rows writes the rows that stay:
// those above it, and of those equal to it the first ones, counted by a scan.  Reads the weights four times, from HBM once.
//
// Moving (gqa_move_kernel): row kept[j] goes to row j <= kept[j], in place, read once and written once.  A workgroup takes a segment of
// rows of one head of K or of V, loads all its sources into registers, says so in a flag, waits until the rows it is about to overwrite have been
// read -- their readers are segments in front of it, two at most -- and stores.  Nothing is ever read that was written in this launch, so the
// flags order reads before writes and carry no data.  Segments are numbered by a ticket as workgroups start, and a workgroup raises its flag
// before it waits: every flag it waits for belongs to one that is running already, whatever the order of dispatch.

#include "mla_common.hpp"
#include "../../include/gqa_attn.h"

using namespace mla;

namespace {

constexpr int PAGE = MLA_PAGE_TOKENS;
constexpr int SEL_THREADS = 1024, SEL_PER = 8, SEL_RUNS = 4, SEL_CHUNK = SEL_THREADS * SEL_PER * SEL_RUNS;
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
    unsigned * sync; int n_sync;                      // ticket and flags of the move, cleared by the selection
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
    __shared__ int      part[SEL_RUNS][16];
    __shared__ unsigned sh_digit;
    __shared__ int      sh_left;
    const int b = blockIdx.x / p.n_head_kv, h = blockIdx.x - b * p.n_head_kv;
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const int n = len_of(p, b), m = min(n, p.n_keep);
    const float * w  = (const float *) (p.w + (int64_t) b * p.w_nb2 + (int64_t) h * p.w_nb1);
    float *       wd = (float *) (p.wd + (int64_t) b * p.wd_nb2 + (int64_t) h * p.wd_nb1);
    int32_t *     kept = p.kept + (int64_t) blockIdx.x * p.n_keep;
    if (h == 0 && tid == 0) p.new_lens[b] = m;
    for (int i = blockIdx.x * SEL_THREADS + tid; i < p.n_sync; i += gridDim.x * SEL_THREADS) p.sync[i] = 0u;
    if (n <= p.n_keep) {                                           // nothing leaves
        for (int i = tid; i < p.n_keep; i += SEL_THREADS) kept[i] = i < n ? i : -1;
        for (int64_t i = tid; i < p.cap; i += SEL_THREADS) wd[i] = i < n ? w[i] : 0.f;
        return;
    }
    const int  c0 = p.n_sink, c1 = n - p.n_recent;                 // the rows that compete (c0 < c1: n_sink + n_recent <= n_keep < n)
    const int  places = p.n_keep - p.n_sink - p.n_recent;
    const bool vec = ((uintptr_t) w & 15) == 0;
    // A chunk: 4 runs of 8192 rows, 8 consecutive ones a thread in each.  All its loads are under way at once, and a sequence of one chunk
    // (32768 rows) is read once: its rows stay in registers over the passes.
    float x[SEL_RUNS][SEL_PER];
    int   held = -1;
    auto load = [&](int base) {
        if (base == held) return;
        held = base;
#pragma unroll
        for (int g = 0; g < SEL_RUNS; g++) {
            const int i0 = base + (g * SEL_THREADS + tid) * SEL_PER;       // rows past the length: nothing is read
            if (vec && i0 + SEL_PER <= n) {
                const f32x4 a = *(const f32x4 *) (w + i0), c = *(const f32x4 *) (w + i0 + 4);
#pragma unroll
                for (int e = 0; e < 4; e++) { x[g][e] = a[e]; x[g][4 + e] = c[e]; }
            } else if (base + g * SEL_THREADS * SEL_PER < n) {
#pragma unroll
                for (int e = 0; e < SEL_PER; e++) x[g][e] = i0 + e < n ? w[i0 + e] : 0.f;
            }
        }
    };

    unsigned prefix = 0;                                           // the digits found so far
    int      left = places;                                        // rows still to be taken among those that share them
    if (places > 0) {
        for (int pass = 0; pass < 3; pass++) {
            const int shift = pass == 0 ? 21 : pass == 1 ? 10 : 0, bits = pass == 2 ? 10 : 11;
            for (int i = tid; i < BINS; i += SEL_THREADS) hist[i] = 0;
            __syncthreads();
            for (int base = 0; base < c1; base += SEL_CHUNK) {
                load(base);
#pragma unroll
                for (int g = 0; g < SEL_RUNS; g++) {
                    const int i0 = base + (g * SEL_THREADS + tid) * SEL_PER;
                    if (base + g * SEL_THREADS * SEL_PER >= c1) continue;
#pragma unroll
                    for (int e = 0; e < SEL_PER; e++) {
                        const int i = i0 + e;
                        const unsigned k = key_of(x[g][e]);
                        if (i >= c0 && i < c1 && (pass == 0 || (k >> (shift + bits)) == prefix)) atomicAdd(&hist[(k >> shift) & ((1u << bits) - 1)], 1u);
                    }
                }
            }
            __syncthreads();
            // the digit at which the rows from the top on reach `left`: thread t holds bins 2047 - 2t and 2046 - 2t
            const int hi = (int) hist[BINS - 1 - 2 * tid], lo = (int) hist[BINS - 2 - 2 * tid];
            int incl = scan_wave(hi + lo, lane);
            if (lane == 63) part[0][wave] = incl;
            __syncthreads();
            for (int q = 0; q < wave; q++) incl += part[0][q];
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
    int taken = 0, ties = 0;                                       // rows before this run: surely kept, and equal to the smallest
    for (int base = 0; base < n; base += SEL_CHUNK) {
        load(base);
        int sure[SEL_RUNS], tie[SEL_RUNS], incl[SEL_RUNS];         // bit e: row 8 (..) + e of the run
#pragma unroll
        for (int g = 0; g < SEL_RUNS; g++) {
            sure[g] = tie[g] = 0;
#pragma unroll
            for (int e = 0; e < SEL_PER; e++) {
                const int i = base + (g * SEL_THREADS + tid) * SEL_PER + e;
                if (i >= n) continue;
                const unsigned k = key_of(x[g][e]);
                if (i < c0 || i >= c1 || (places > 0 && k > prefix)) sure[g] |= 1 << e;
                else if (places > 0 && k == prefix) tie[g] |= 1 << e;
            }
            incl[g] = scan_wave(__popc(sure[g]) | (__popc(tie[g]) << 16), lane);     // (at most 8192 of either in a run)
            if (lane == 63) part[g][wave] = incl[g];
        }
        __syncthreads();                                           // (also: every row of the chunk has been read before one is overwritten)
#pragma unroll
        for (int g = 0; g < SEL_RUNS; g++) {
            if (base + g * SEL_THREADS * SEL_PER >= n) continue;
            int before = incl[g] - (__popc(sure[g]) | (__popc(tie[g]) << 16)), all = 0;
            for (int q = 0; q < 16; q++) { if (q < wave) before += part[g][q]; all += part[g][q]; }
            int s = taken + (before & 0xffff), t = ties + (before >> 16);
#pragma unroll
            for (int e = 0; e < SEL_PER; e++) {
                const bool is_sure = sure[g] >> e & 1, is_tie = tie[g] >> e & 1;
                if (is_sure || (is_tie && t < left)) {
                    const int j = s + min(t, left);
                    kept[j] = base + (g * SEL_THREADS + tid) * SEL_PER + e;
                    wd[j]   = x[g][e];
                }
                s += is_sure; t += is_tie;
            }
            taken += all & 0xffff; ties += all >> 16;
        }
        __syncthreads();
    }
    for (int64_t i = p.n_keep + tid; i < p.cap; i += SEL_THREADS) wd[i] = 0.f;
}

constexpr int MOVE_THREADS = 512, MOVE_R = 12, MOVE_UNITS = MOVE_THREADS * MOVE_R;     // units a workgroup holds in registers: 96 KB of 16 bytes each
constexpr int MOVE_SEGMENTS = 63 * MOVE_THREADS;                                        // of a head: a bit of a thread each

// The segments of one kind of rows (K or V): `rows` of them a segment, `magic` = ceil(2^32 / units): f / units = f * magic >> 32 for f < MOVE_UNITS.
struct Seg { int units, rows, count; unsigned magic; };

template <typename T>
__global__ void __launch_bounds__(MOVE_THREADS) gqa_move_kernel(const EvictP p, const Seg sk, const Seg sv, unsigned * sync) {
    __shared__ unsigned sh_ticket;
    if (threadIdx.x == 0) sh_ticket = __hip_atomic_fetch_add(sync, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    __syncthreads();
    // in tickets, every group's first segment comes before any group's second, K before V
    const unsigned groups = (unsigned) (p.n_seq * p.n_head_kv), n_k = groups * (unsigned) sk.count;
    const bool     is_k = sh_ticket < n_k;
    const unsigned t = is_k ? sh_ticket : sh_ticket - n_k;
    const int      seg = (int) (t / groups), group = (int) (t - (unsigned) seg * groups);
    const Seg      sg = is_k ? sk : sv;
    const int      b = group / p.n_head_kv, h = group - b * p.n_head_kv;
    if (len_of(p, b) <= p.n_keep) return;                          // (the whole group returns: nobody waits for it)
    unsigned *     flags = sync + 1 + (is_k ? 0 : n_k) + (unsigned) group * (unsigned) sg.count;
    char *         base = is_k ? p.k + h * p.k_head : p.v + h * p.v_head;
    const int64_t  nb_page = is_k ? p.k_page : p.v_page, nb_row = is_k ? p.k_row : p.v_row;
    const int32_t * kept = p.kept + (int64_t) group * p.n_keep;
    const int32_t * bt = p.block_table + (int64_t) b * p.bt_stride;
    const int      j0 = seg * sg.rows, j1 = min(j0 + sg.rows, p.n_keep), last = j1 - 1;

    T        x[MOVE_R];
    unsigned moves = 0;                                            // bit r: the row has another place, and both have memory
    int      src[MOVE_R], from[MOVE_R], into[MOVE_R];
#pragma unroll
    for (int r = 0; r < MOVE_R; r++) src[r] = kept[min(j0 + (int) __umulhi(r * MOVE_THREADS + threadIdx.x, sg.magic), last)];
    // segments in front that read rows this one overwrites: bit k of thread t is segment t + 512 k (kept rises, so a segment reads a range)
    uint64_t readers = 0;
    for (int k = 0, s = (int) threadIdx.x; s < seg; k++, s += MOVE_THREADS)
        readers |= (uint64_t) ((int) (kept[s * sg.rows] < j1) & (int) (kept[(s + 1) * sg.rows - 1] >= j0)) << k;
#pragma unroll
    for (int r = 0; r < MOVE_R; r++) {
        from[r] = bt[src[r] / PAGE];
        into[r] = bt[min(j0 + (int) __umulhi(r * MOVE_THREADS + threadIdx.x, sg.magic), last) / PAGE];
    }
#pragma unroll
    for (int r = 0; r < MOVE_R; r++) {                             // (no && in here: a branch would put a wait between the loads)
        const int f = r * MOVE_THREADS + (int) threadIdx.x, row = (int) __umulhi(f, sg.magic), j = j0 + row, unit = f - row * sg.units;
        const int go = (int) (j <= last) & (int) (src[r] != j) & (int) (from[r] >= 0) & (int) (from[r] < p.n_pages) & (int) (into[r] >= 0) & (int) (into[r] < p.n_pages);
        // rows that stay: page 0 of the pool, always there
        x[r] = *(const T *) (base + (go ? from[r] * nb_page + (src[r] % PAGE) * nb_row + unit * (int) sizeof(T) : 0));
        moves |= (unsigned) go << r;
    }
    // every source is in a register before the flag goes up
#pragma unroll
    for (int r = 0; r < MOVE_R; r++) asm volatile("" : "+v"(x[r]) :: "memory");
    __syncthreads();
    if (threadIdx.x == 0) __hip_atomic_store(flags + seg, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    for (int k = 0, s = (int) threadIdx.x; readers >> k; k++, s += MOVE_THREADS)
        if (readers >> k & 1)
            while (__hip_atomic_load(flags + s, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) == 0u) __builtin_amdgcn_s_sleep(1);
    __syncthreads();
#pragma unroll
    for (int r = 0; r < MOVE_R; r++) {
        const int f = r * MOVE_THREADS + (int) threadIdx.x, row = (int) __umulhi(f, sg.magic), j = j0 + row, unit = f - row * sg.units;
        if (moves >> r & 1) *(T *) (base + into[r] * nb_page + (j % PAGE) * nb_row + unit * (int) sizeof(T)) = x[r];
    }
}

int check_pool(const gqa_pool & c, int row_bytes) {
    if (!c.data) return MLA_ERR_NULL;
    if (((uintptr_t) c.data & 3) || (c.nb_page & 3) || (c.nb_row & 3) || (c.nb_head & 3) || (row_bytes & 3)) return MLA_ERR_BAD_ALIGNMENT;
    return c.nb_page < 0 || c.nb_row < 0 || c.nb_head < 0 || row_bytes < 8 || row_bytes > (1 << 14) ? MLA_ERR_BAD_SHAPE : 0;
}
bool wide(const gqa_pool & c, int row_bytes) { return row_bytes >= 32 && !(((uintptr_t) c.data & 15) || (c.nb_page & 15) || (c.nb_row & 15) || (c.nb_head & 15) || (row_bytes & 15)); }

Seg make_seg(int row_bytes, int unit, int64_t n_keep) {
    Seg s;
    s.units = row_bytes / unit;
    s.rows  = MOVE_UNITS / s.units;
    s.count = (int) ((n_keep + s.rows - 1) / s.rows);
    s.magic = (unsigned) ((((uint64_t) 1 << 32) + s.units - 1) / s.units);     // (two units a row at least: 2^32 would not fit)
    return s;
}

struct Plan {
    bool    w16;              // units of 16 bytes, else of 4
    Seg     k, v;
    int64_t segments;         // of all heads, K and V
    size_t  bytes;            // of the workspace: the ticket and a flag a segment
};

Plan make_plan(const gqa_evict_args * a) {
    Plan pl;
    pl.w16 = wide(a->k, a->k_row_bytes) && (!a->v.data || wide(a->v, a->v_row_bytes));
    const int64_t cap = a->bt_stride * PAGE, n_keep = a->n_keep < cap ? a->n_keep : 0;     // (a table no wider than n_keep holds nothing to evict)
    pl.k = make_seg(a->k_row_bytes, pl.w16 ? 16 : 4, n_keep);
    pl.v = a->v.data ? make_seg(a->v_row_bytes, pl.w16 ? 16 : 4, n_keep) : Seg{ 1, 1, 0, 0u };
    pl.segments = (int64_t) a->n_seq * a->n_head_kv * (pl.k.count + pl.v.count);
    pl.bytes = (size_t) (1 + pl.segments) * 4;
    return pl;
}

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
    const Plan pl = make_plan(a);
    if (pl.k.count > MOVE_SEGMENTS || pl.v.count > MOVE_SEGMENTS || pl.segments >= ((int64_t) 1 << 30)) return MLA_ERR_BAD_SHAPE;
    return 0;
}

extern "C" size_t gqa_evict_workspace_size(const gqa_evict_args * a) {
    if (gqa_evict_check(a) || a->n_seq == 0) return 0;
    return make_plan(a).bytes;
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
    const Plan pl = make_plan(a);
    if (!a->workspace || ((uintptr_t) a->workspace & 255) || a->workspace_size < pl.bytes) return MLA_ERR_WORKSPACE;
    const unsigned groups = (unsigned) (a->n_seq * a->n_head_kv);
    p.sync = (unsigned *) a->workspace; p.n_sync = (int) (1 + pl.segments);
    hipLaunchKernelGGL(gqa_select_kernel, dim3(groups), dim3(SEL_THREADS), 0, (hipStream_t) stream, p);
    hipError_t e = hipGetLastError();
    if (e != hipSuccess) return (int) e;
    if (pl.segments == 0) return 0;
    if (pl.w16) hipLaunchKernelGGL(gqa_move_kernel<u32x4>, dim3((unsigned) pl.segments), dim3(MOVE_THREADS), 0, (hipStream_t) stream, p, pl.k, pl.v, p.sync);
    else        hipLaunchKernelGGL(gqa_move_kernel<unsigned>, dim3((unsigned) pl.segments), dim3(MOVE_THREADS), 0, (hipStream_t) stream, p, pl.k, pl.v, p.sync);
    return (int) hipGetLastError();
}
