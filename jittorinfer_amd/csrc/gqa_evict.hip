// Eviction from a paged cache by accumulated attention weight (include/gqa_attn.h), for gfx950: which rows stay, and their way up.
//
// Selection (gqa_select_kernel, a workgroup per (sequence, KV head)): the weights' bits, made monotone, are searched digit by digit for the
// smallest weight that stays (11 + 11 + 10 bits, a histogram in LDS each), then one pass in the order of the rows writes the rows that stay:
// those above it, and of those equal to it the first ones, counted by a scan.  Bound by its chain of passes and barriers, not by bytes: 12.1 us for 8
// groups of 8192 rows, 14.3 for 256.  Block tables of more rows take several workgroups a group (gqa_rank_kernel: 26 us for 100000 rows, 93 in one).
//
// Moving (gqa_move_kernel): row kept[j] goes to row j <= kept[j], in place, read once and written once.  A workgroup takes a segment of
// rows of one head of K or of V, loads all its sources into registers, says so in a flag, waits until the rows it is about to overwrite have been
// read -- their readers are segments in front of it, two at most -- and stores.  Nothing is ever read that was written in this launch, so the
// flags order reads before writes and carry no data.  Segments are numbered by a ticket as workgroups start, and a workgroup raises its flag
// before it waits: every flag it waits for belongs to one that is running already, whatever the order of dispatch.  Bound by HBM where there is
// much to move: 32 sequences of 8 heads cut from up to 8192 rows to 2048, 479 MB read and written in 106 us = 4.5 TB/s (a large copy: 4.9); two latent
// caches cut from 100000 rows to 40000 41 us; 8192 rows of one sequence to 4096 12.2 us.  (A workgroup a stripe of columns, all rows in
// order, needed no flags and took 234 us for the second: 36 workgroups cannot keep enough loads under way.)

#include "gqa_common.hpp"

using namespace mla;
using namespace mla::gqa;

namespace {

constexpr int SEL_THREADS = 1024, SEL_PER = 8, SEL_RUN = SEL_THREADS * SEL_PER, SEL_RUNS = 4, SEL_CHUNK = SEL_RUN * SEL_RUNS;
// One workgroup a group, or one a run of 8192 rows in four launches.  Measured, a whole call: 8 groups of 16384 rows 24.9 against 32.3 us, of 32768
// rows 36.9 against 34.0; 64 groups of 32768 rows 53.4 against 55.5, of 131072 190 against 169; 256 groups of 65536 rows 293 against 344.
constexpr int SEL_ONE = 3 * SEL_RUN, SEL_GROUPS = 64, SEL_MANY = 8192;       // (SEL_MANY runs at most: 128 MB of histograms)
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

// The digit at which the rows of a histogram, counted from the largest digit down, reach `left`, and how many of the digit's own rows those are.
// One wave: lane t sums the 32 bins 2047 - 32 t and down (rotated, so that the lanes meet different banks), a scan finds the lane, another the bin.
struct Pick { unsigned digit; int left; };
__device__ __forceinline__ Pick pick(const unsigned * hist, int left, int lane) {
    int sum = 0;
#pragma unroll
    for (int i = 0; i < 32; i++) sum += (int) hist[BINS - 1 - 32 * lane - ((i + lane) & 31)];
    const int incl = scan_wave(sum);
    const int at   = __ffsll(__ballot(incl - sum < left && incl >= left)) - 1;
    const int base = lane_of(incl - sum, at);
    const int bin  = BINS - 1 - 32 * at - (lane & 31);
    const int mine = lane < 32 ? (int) hist[bin] : 0;
    const int upto = base + scan_wave(mine);
    const int win  = __ffsll(__ballot(lane < 32 && upto - mine < left && upto >= left)) - 1;
    return Pick{ (unsigned) lane_of(bin, win), left - lane_of(upto - mine, win) };
}

// Digits of a key, from the top: 11, 11 and 10 bits.
__device__ __forceinline__ constexpr int shift_of(int pass) { return pass == 0 ? 21 : pass == 1 ? 10 : 0; }
__device__ __forceinline__ constexpr int bits_of(int pass) { return pass == 2 ? 10 : 11; }

// What a (sequence, KV head) has to decide.
struct Group {
    int n, c0, c1, places;                                         // rows; those that compete: [c0, c1), for so many places
    const float * w; float * wd; int32_t * kept;
};
__device__ __forceinline__ Group group_of(const EvictP & p, int group) {
    Group g;
    const int b = group / p.n_head_kv, h = group - b * p.n_head_kv;
    g.n  = len_of(p, b);
    g.c0 = p.n_sink; g.c1 = g.n - p.n_recent;                      // (c0 < c1 where rows leave: n_sink + n_recent <= n_keep < n)
    g.places = p.n_keep - p.n_sink - p.n_recent;
    g.w  = (const float *) (p.w + (int64_t) b * p.w_nb2 + (int64_t) h * p.w_nb1);
    g.wd = (float *) (p.wd + (int64_t) b * p.wd_nb2 + (int64_t) h * p.wd_nb1);
    g.kept = p.kept + (int64_t) group * p.n_keep;
    return g;
}

// 8 rows from i0 on; past the length nothing is read.
__device__ __forceinline__ void load_rows(const Group & g, int i0, float (&x)[SEL_PER]) {
    if (((uintptr_t) g.w & 15) == 0 && i0 + SEL_PER <= g.n) {
        const f32x4 a = *(const f32x4 *) (g.w + i0), c = *(const f32x4 *) (g.w + i0 + 4);
#pragma unroll
        for (int e = 0; e < 4; e++) { x[e] = a[e]; x[4 + e] = c[e]; }
    } else {
#pragma unroll
        for (int e = 0; e < SEL_PER; e++) x[e] = i0 + e < g.n ? g.w[i0 + e] : 0.f;
    }
}
__device__ __forceinline__ void count_rows(const Group & g, int i0, const float (&x)[SEL_PER], int pass, unsigned prefix, unsigned * hist) {
#pragma unroll
    for (int e = 0; e < SEL_PER; e++) {
        const unsigned k = key_of(x[e]);
        if (i0 + e >= g.c0 && i0 + e < g.c1 && (pass == 0 || (k >> (shift_of(pass) + bits_of(pass))) == prefix))
            atomicAdd(&hist[(k >> shift_of(pass)) & ((1u << bits_of(pass)) - 1)], 1u);
    }
}
// The 8 rows are in registers before anything that follows (a barrier, or a flag, that lets others overwrite them): the compiler may otherwise leave a load under
// way whose number it needs last.
__device__ __forceinline__ void pin_rows(float (&x)[SEL_PER]) {
#pragma unroll
    for (int e = 0; e < SEL_PER; e++) asm volatile("" : "+v"(x[e]) :: "memory");
}
// Of 8 rows: those that stay whatever the others do (bits 0 .. 7), and those equal to the smallest weight that stays, `last` (bits 16 ..).
__device__ __forceinline__ unsigned sort_rows(const Group & g, int i0, const float (&x)[SEL_PER], unsigned last) {
    unsigned m = 0;
#pragma unroll
    for (int e = 0; e < SEL_PER; e++) {
        const int i = i0 + e;
        const unsigned k = key_of(x[e]);
        const bool in = i < g.n, held = i < g.c0 || i >= g.c1;
        if (in && (held || (g.places > 0 && k > last))) m |= 1u << e;
        else if (in && g.places > 0 && k == last) m |= 0x10000u << e;
    }
    return m;
}
__device__ __forceinline__ int count_both(unsigned m) { return __popc(m & 0xffffu) | (__popc(m >> 16) << 16); }
// Writes them out: `sure` rows kept for certain and `ties` equal ones come before these 8.
__device__ __forceinline__ void place_rows(const Group & g, int i0, const float (&x)[SEL_PER], unsigned m, int sure, int ties, int left) {
#pragma unroll
    for (int e = 0; e < SEL_PER; e++) {
        const bool is_sure = m >> e & 1, is_tie = m >> (16 + e) & 1;
        if (is_sure || (is_tie && ties < left)) {
            const int j = sure + min(ties, left);
            g.kept[j] = i0 + e;
            g.wd[j]   = x[e];
        }
        sure += is_sure; ties += is_tie;
    }
}

// One workgroup a group.
__global__ void __launch_bounds__(SEL_THREADS) gqa_select_kernel(const EvictP p) {
    __shared__ unsigned hist[2][BINS];
    __shared__ int      part[SEL_RUNS][16];
    __shared__ Pick     sh_pick;
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const Group g = group_of(p, blockIdx.x);
    if (blockIdx.x % p.n_head_kv == 0 && tid == 0) p.new_lens[blockIdx.x / p.n_head_kv] = min(g.n, p.n_keep);
    for (int i = blockIdx.x * SEL_THREADS + tid; i < p.n_sync; i += gridDim.x * SEL_THREADS) p.sync[i] = 0u;
    if (g.n <= p.n_keep) {                                         // nothing leaves
        for (int64_t i = tid; i < p.n_keep; i += SEL_THREADS) g.kept[i] = i < g.n ? (int) i : -1;      // (n_keep up to 2^31 - 1)
        for (int64_t i = tid; i < p.cap; i += SEL_THREADS) g.wd[i] = i < g.n ? g.w[i] : 0.f;
        return;
    }
    // A chunk: 4 runs of 8192 rows, 8 consecutive ones a thread in each.  All its loads are under way at once, and a sequence of one chunk
    // (32768 rows) is read once: its rows stay in registers over the passes.
    float x[SEL_RUNS][SEL_PER];
    int   held = -1;
    auto load = [&](int base) {
        if (base == held) return;
        held = base;
#pragma unroll
        for (int r = 0; r < SEL_RUNS; r++) if (base + r * SEL_RUN < g.n) load_rows(g, base + r * SEL_RUN + tid * SEL_PER, x[r]);
    };
    Pick got{ 0u, g.places };                                      // the digits found so far; rows still to be taken among those that share them
    if (g.places > 0) {
        hist[0][2 * tid] = hist[0][2 * tid + 1] = 0u;
        load(0);
        __syncthreads();
#pragma unroll
        for (int pass = 0; pass < 3; pass++) {
            unsigned * now = hist[pass & 1], * next = hist[(pass & 1) ^ 1];
            for (int base = 0; base < g.c1; base += SEL_CHUNK) {
                load(base);
#pragma unroll
                for (int r = 0; r < SEL_RUNS; r++) if (base + r * SEL_RUN < g.c1) count_rows(g, base + r * SEL_RUN + tid * SEL_PER, x[r], pass, got.digit, now);
            }
            next[2 * tid] = next[2 * tid + 1] = 0u;
            __syncthreads();
            if (wave == 0) {
                const Pick q = pick(now, got.left, lane);
                if (lane == 0) sh_pick = q;
            }
            __syncthreads();
            got.digit = (got.digit << bits_of(pass)) | sh_pick.digit;
            got.left  = sh_pick.left;
        }
    }
    // got: the key of the smallest weight that stays, and how many rows of it do
    int sure = 0, ties = 0;                                        // rows before this run
    for (int base = 0; base < g.n; base += SEL_CHUNK) {
        load(base);
        unsigned m[SEL_RUNS];
        int      incl[SEL_RUNS];
#pragma unroll
        for (int r = 0; r < SEL_RUNS; r++) {
            m[r] = base + r * SEL_RUN < g.n ? sort_rows(g, base + r * SEL_RUN + tid * SEL_PER, x[r], got.digit) : 0u;
            incl[r] = scan_wave(count_both(m[r]));           // (at most 8192 of either in a run)
            if (lane == 63) part[r][wave] = incl[r];
            if (base + r * SEL_RUN < g.n) pin_rows(x[r]);
        }
        __syncthreads();                                           // (also: every row of the chunk has been read before one is overwritten)
#pragma unroll
        for (int r = 0; r < SEL_RUNS; r++) {
            if (base + r * SEL_RUN >= g.n) continue;
            const int upto = scan_wave(lane < 16 ? part[r][lane] : 0);
            const int all = lane_of(upto, 15), ahead = wave ? lane_of(upto, wave - 1) : 0;
            const int before = ahead + incl[r] - count_both(m[r]);
            place_rows(g, base + r * SEL_RUN + tid * SEL_PER, x[r], m[r], sure + (before & 0xffff), ties + (before >> 16), got.left);
            sure += all & 0xffff; ties += all >> 16;
        }
        __syncthreads();
    }
    for (int64_t i = p.n_keep + tid; i < p.cap; i += SEL_THREADS) g.wd[i] = 0.f;
}

// The same over several workgroups a group, a run of 8192 rows each, in four launches: PASS 0, 1, 2 leave every run's histogram of a digit,
// PASS 1, 2, 3 add up those of the pass before and pick its digit, each workgroup for itself.  PASS 3 writes the rows that stay, behind those of the
// runs in front: every run publishes its two counts (in one word, that is its flag too) and waits for the words of the runs before it; runs are
// numbered by a ticket and publish before they wait, so they wait for running workgroups only.
struct Rank { unsigned * hist; uint64_t * counts; Pick * picks; unsigned * ticket; int runs; };   // hist [2][groups][runs][BINS], counts [groups][runs], picks [groups][2]

template <int PASS>
__global__ void __launch_bounds__(SEL_THREADS) gqa_rank_kernel(const EvictP p, const Rank k) {
    __shared__ unsigned hist[BINS];
    __shared__ int      part[16];
    __shared__ Pick     sh_pick;
    __shared__ unsigned sh_ticket;
    __shared__ unsigned long long sh_before;
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int groups = p.n_seq * p.n_head_kv;
    int number = (int) blockIdx.x;
    if constexpr (PASS == 0) {
        for (int i = blockIdx.x * SEL_THREADS + tid; i < p.n_sync; i += gridDim.x * SEL_THREADS) p.sync[i] = 0u;
        if (tid == 0) k.counts[blockIdx.x] = 0;
        if (blockIdx.x == 0 && tid == 0) *k.ticket = 0u;
    }
    if constexpr (PASS == 3) {
        if (tid == 0) { sh_ticket = __hip_atomic_fetch_add(k.ticket, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT); sh_before = 0; }
        __syncthreads();
        number = (int) sh_ticket;
    }
    const int   run = number / groups, group = number - run * groups;      // a group's first run before any group's second
    const Group g = group_of(p, group);
    const int   i0 = run * SEL_RUN + tid * SEL_PER;
    if constexpr (PASS < 3) {
        if (g.n <= p.n_keep || g.places == 0) return;
    } else {
        if (run == 0 && group % p.n_head_kv == 0 && tid == 0) p.new_lens[group / p.n_head_kv] = min(g.n, p.n_keep);
        if (g.n <= p.n_keep) {
            const int64_t end = run == k.runs - 1 ? (p.cap > p.n_keep ? p.cap : p.n_keep) : (int64_t) (run + 1) * SEL_RUN;
            for (int64_t i = (int64_t) run * SEL_RUN + tid; i < end; i += SEL_THREADS) {
                if (i < p.n_keep) g.kept[i] = i < g.n ? (int) i : -1;
                if (i < p.cap) g.wd[i] = i < g.n ? g.w[i] : 0.f;
            }
            return;
        }
    }
    float x[SEL_PER];
    load_rows(g, i0, x);
    Pick got{ 0u, g.places };
    if (PASS > 0 && g.places > 0) {
        const unsigned * from = k.hist + ((size_t) ((PASS - 1) & 1) * groups + group) * k.runs * BINS;
        const int        live = min(k.runs, (g.c1 + SEL_RUN - 1) / SEL_RUN);
        unsigned a = 0, c = 0;
        for (int r0 = 0; r0 < live; r0 += 8) {                     // 16 loads under way at a time
            unsigned v[16];
#pragma unroll
            for (int r = 0; r < 8; r++) {
                const unsigned * row = from + (size_t) min(r0 + r, live - 1) * BINS + tid;
                v[2 * r] = row[0]; v[2 * r + 1] = row[SEL_THREADS];
            }
#pragma unroll
            for (int r = 0; r < 8; r++) if (r0 + r < live) { a += v[2 * r]; c += v[2 * r + 1]; }
        }
        hist[tid] = a; hist[SEL_THREADS + tid] = c;
        if constexpr (PASS > 1) got = k.picks[group * 2 + (PASS & 1)];      // the pass before's: digits but the last
        __syncthreads();
        if (wave == 0) {
            const Pick q = pick(hist, got.left, lane);
            if (lane == 0) sh_pick = q;
        }
        __syncthreads();
        got.digit = (got.digit << bits_of(PASS - 1)) | sh_pick.digit;
        got.left  = sh_pick.left;
        if (PASS < 3 && run == 0 && tid == 0) k.picks[group * 2 + ((PASS + 1) & 1)] = got;
    }
    if constexpr (PASS < 3) {
        if (run * SEL_RUN >= g.c1) return;
        hist[tid] = hist[SEL_THREADS + tid] = 0u;
        __syncthreads();
        count_rows(g, i0, x, PASS, got.digit, hist);
        __syncthreads();
        unsigned * to = k.hist + (((size_t) (PASS & 1) * groups + group) * k.runs + run) * BINS;
        to[tid] = hist[tid]; to[SEL_THREADS + tid] = hist[SEL_THREADS + tid];
    } else {
        const unsigned m = sort_rows(g, i0, x, got.digit);
        const int incl = scan_wave(count_both(m));
        if (lane == 63) part[wave] = incl;
        pin_rows(x);
        __syncthreads();                                           // (every row of the run is in a register: it may be overwritten from here on)
        const int upto = scan_wave(lane < 16 ? part[lane] : 0);
        const int all = lane_of(upto, 15), ahead = wave ? lane_of(upto, wave - 1) : 0;
        uint64_t * counts = k.counts + (size_t) group * k.runs;
        if (tid == 0) __hip_atomic_store(counts + run, (uint64_t) 1 << 63 | (uint64_t) (all >> 16) << 31 | (uint64_t) (all & 0xffff), __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        for (int r = tid; r < run; r += SEL_THREADS) {             // (sums below 2^31 in each half)
            uint64_t v;
            while (!((v = __hip_atomic_load(counts + r, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT)) >> 63)) __builtin_amdgcn_s_sleep(1);
            atomicAdd(&sh_before, (unsigned long long) (v << 1 >> 1));
        }
        __syncthreads();
        const int sure = (int) (sh_before & 0x7fffffffu), ties = (int) (sh_before >> 31);
        const int before = ahead + incl - count_both(m);
        place_rows(g, i0, x, m, sure + (before & 0xffff), ties + (before >> 16), got.left);
        const int64_t end = min((int64_t) (run + 1) * SEL_RUN, p.cap);      // the run's own share of the rows past the new length
        for (int64_t i = max((int64_t) run * SEL_RUN, (int64_t) p.n_keep) + tid; i < end; i += SEL_THREADS) g.wd[i] = 0.f;
    }
}

constexpr int MOVE_THREADS = 512, MOVE_R = 12, MOVE_UNITS = MOVE_THREADS * MOVE_R;     // units a workgroup holds in registers: 96 KB of 16 bytes each

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
    // Segments in front that may read rows this one overwrites: kept rises, so each of them reads from a range of its own at least as long as the rows it moves,
    // as many as are overwritten here at least; two such ranges at most, side by side, reach into [j0, j1).  So a thread meets one at most: it looks at every 512th.
    int reader = -1;
    for (int s = (int) threadIdx.x; s < seg; s += MOVE_THREADS)
        reader = (int) (kept[s * sg.rows] < j1) & (int) (kept[(s + 1) * sg.rows - 1] >= j0) ? s : reader;
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
    if (reader >= 0)
        while (__hip_atomic_load(flags + reader, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) == 0u) __builtin_amdgcn_s_sleep(1);
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
    int     runs;             // of the selection over several workgroups; 0: one
    size_t  off_ticket, off_counts, off_picks, off_hist, bytes;    // of the workspace: the move's ticket and a flag a segment come first
};

Plan make_plan(const gqa_evict_args * a) {
    Plan pl;
    pl.w16 = wide(a->k, a->k_row_bytes) && (!a->v.data || wide(a->v, a->v_row_bytes));
    const int64_t cap = a->bt_stride * PAGE, n_keep = a->n_keep < cap ? a->n_keep : 0;     // (a table no wider than n_keep holds nothing to evict)
    pl.k = make_seg(a->k_row_bytes, pl.w16 ? 16 : 4, n_keep);
    pl.v = a->v.data ? make_seg(a->v_row_bytes, pl.w16 ? 16 : 4, n_keep) : Seg{ 1, 1, 0, 0u };
    pl.segments = (int64_t) a->n_seq * a->n_head_kv * (pl.k.count + pl.v.count);
    const size_t groups = (size_t) a->n_seq * a->n_head_kv;
    const int64_t runs = (cap + SEL_RUN - 1) / SEL_RUN;
    pl.runs = cap > SEL_ONE && n_keep && groups <= SEL_GROUPS && (int64_t) groups * runs <= SEL_MANY ? (int) runs : 0;
    size_t at = 0;
    auto take = [&](size_t n) { const size_t o = at; at += (n + 255) & ~(size_t) 255; return o; };
    take((size_t) (1 + pl.segments) * 4);
    pl.off_ticket = take(4);
    pl.off_counts = take(groups * pl.runs * 8);
    pl.off_picks  = take(groups * 2 * sizeof(Pick));
    pl.off_hist   = take(groups * 2 * pl.runs * BINS * 4);
    pl.bytes = at;
    return pl;
}

}  // namespace

extern "C" int gqa_evict_check(const gqa_evict_args * a) {
    if (!a) return MLA_ERR_NULL;
    if (a->n_seq < 0 || a->n_head_kv < 1 || a->n_keep < 1 || a->n_sink < 0 || a->n_recent < 0 || (int64_t) a->n_sink + a->n_recent > a->n_keep) return MLA_ERR_BAD_SHAPE;
    if (a->n_seq == 0) return 0;
    if (!a->weights || !a->weights_dst || !a->kept || !a->new_lens || !a->block_table || !a->seq_lens) return MLA_ERR_NULL;
    if (a->n_pages < 1 || a->bt_stride < 1 || a->bt_stride >= ((int64_t) 1 << 30) / PAGE || (int64_t) a->n_seq * a->n_head_kv > 65535) return MLA_ERR_BAD_SHAPE;
    int rc = check_pool(a->k, a->k_row_bytes);
    if (!rc && a->v.data) rc = check_pool(a->v, a->v_row_bytes);
    if (rc) return rc;
    if (((uintptr_t) a->weights & 3) || (a->w_nb1 & 3) || (a->w_nb2 & 3) || ((uintptr_t) a->weights_dst & 3) || (a->wd_nb1 & 3) || (a->wd_nb2 & 3)) return MLA_ERR_BAD_ALIGNMENT;
    if (a->weights == a->weights_dst && (a->w_nb1 != a->wd_nb1 || a->w_nb2 != a->wd_nb2)) return MLA_ERR_BAD_SHAPE;
    if (a->new_lens == a->seq_lens || a->v.data == a->k.data) return MLA_ERR_UNSUPPORTED;
    const int64_t apart = (const char *) a->weights_dst - (const char *) a->weights, row = a->bt_stride * PAGE * 4;
    if (apart && apart > -row && apart < row) return MLA_ERR_UNSUPPORTED;
    const Plan pl = make_plan(a);
    // (a launch holds fewer than 2^32 threads)
    if (pl.segments >= ((int64_t) 1 << 32) / MOVE_THREADS) return MLA_ERR_BAD_SHAPE;
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
    if (pl.runs) {
        char * ws = (char *) a->workspace;
        const Rank k{ (unsigned *) (ws + pl.off_hist), (uint64_t *) (ws + pl.off_counts), (Pick *) (ws + pl.off_picks), (unsigned *) (ws + pl.off_ticket), pl.runs };
        const dim3 grid(groups * (unsigned) pl.runs);
        hipLaunchKernelGGL(gqa_rank_kernel<0>, grid, dim3(SEL_THREADS), 0, (hipStream_t) stream, p, k);
        hipLaunchKernelGGL(gqa_rank_kernel<1>, grid, dim3(SEL_THREADS), 0, (hipStream_t) stream, p, k);
        hipLaunchKernelGGL(gqa_rank_kernel<2>, grid, dim3(SEL_THREADS), 0, (hipStream_t) stream, p, k);
        hipLaunchKernelGGL(gqa_rank_kernel<3>, grid, dim3(SEL_THREADS), 0, (hipStream_t) stream, p, k);
    } else hipLaunchKernelGGL(gqa_select_kernel, dim3(groups), dim3(SEL_THREADS), 0, (hipStream_t) stream, p);
    hipError_t e = hipGetLastError();
    if (e != hipSuccess) return (int) e;
    if (pl.segments == 0) return 0;
    if (pl.w16) hipLaunchKernelGGL(gqa_move_kernel<u32x4>, dim3((unsigned) pl.segments), dim3(MOVE_THREADS), 0, (hipStream_t) stream, p, pl.k, pl.v, p.sync);
    else        hipLaunchKernelGGL(gqa_move_kernel<unsigned>, dim3((unsigned) pl.segments), dim3(MOVE_THREADS), 0, (hipStream_t) stream, p, pl.k, pl.v, p.sync);
    return (int) hipGetLastError();
}
