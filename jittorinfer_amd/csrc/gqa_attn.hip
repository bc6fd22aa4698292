// Attention of one new token of every sequence over a paged cache of ordinary heads (include/gqa_attn.h), for gfx950.
//
//   o[b, h] = sum_i p_i v_i,  p = softmax_i(scale * q[b, h] . k_i [soft cap] [+ mask]),  i over the sequence's rows of KV head h / G
//
// Every row of K and V is used by G query heads once, 2 G flop a byte: the kernel is bound by the bytes of the cache.  So a wave takes
// its operands from HBM straight into the matrix cores' registers and keeps everything else there, without LDS or a barrier in the
// loop:
//   * a wave owns a tile of 32 rows.  S^T = K Q^T: a 16x16x32 MFMA takes 16 rows of K as they lie in memory (lane (r, g) holds 16 bytes
//     of row r, the four g make 64 consecutive bytes) and leaves in lane (h, g) the scores of head h with rows 4g .. 4g + 3.
//   * those registers, exponentiated, are the A operand of O = P V when contraction index (g, e) stands for row 4g + e of the tile's first 16
//     rows (e < 4) or its last 16: P never leaves the lane that computed it.
//   * V: lane (i, g) loads, of the same 8 rows, the 16 bytes of columns 8i .. 8i + 7: 256 consecutive bytes a row.  An 8 x 8 block of
//     values a lane, transposed in its own registers by v_perm_b32 (half an instruction a value), gives the B operands of 8 MFMAs, the
//     columns {8i + c} one MFMA each.
//   * P goes in as a sum of 16-bit numbers, three of bf16 (24 bits) or two of f16 (22 bits): the matrix cores are idle otherwise, and P
//     rounded to one (2^-9 in bf16) or two of bf16 (2^-17) would be the largest error of the whole pass.
//   * the running maximum moves only when a score passes it by more than 2^8 (2^4 in f16; sums then reach 2^8 a key, far from f32's range), so
//     the common tile has no reduction across lanes and no rescaling.
//   * K of the next tile is requested when this tile's scores are done, V when its products are.
//
// Work: the list of all (sequence, head block, page) units, in that order, is dealt to the workgroups in equal runs, from the lengths on
// the device (nothing on the host depends on them, so a captured launch stays valid while they change).  A run that covers a (sequence,
// head block) whole writes its result; the others leave (o, m, l) in f32 for gqa_join_kernel, which joins them in the order of the rows.
// With weights the first kernel also leaves every score, 4 bytes a (head, row), and gqa_join_kernel adds exp(s - m) / l over the group too.
//
// Measured, 32 query heads on 8 of 128, bf16, a whole call: 32 x 8192 rows 191 us = 5.6 TB/s (head by head 186 = 5.8; a large copy moves 4.9), 64 x 16384
// 748 us = 5.7 (702 = 6.1), 1 x 1024 rows 11.4 us, latency alone: 6.7 of it this kernel, 4.5 the join.

#include <float.h>
#include <limits.h>
#include <math.h>

#include <atomic>
#include <type_traits>

#include "gqa_common.hpp"

using namespace mla;
using namespace mla::gqa;

namespace {

struct AttnP {
    const char * q; int64_t q_nb1, q_nb2; int q_f32;
    const char * k; unsigned k_page; int64_t k_head; int k_row;
    const char * v; unsigned v_page; int64_t v_head; int v_row;
    int64_t n_pages;
    const int32_t * block_table; int64_t bt_stride;
    const int32_t * seq_lens;
    const char * mask; int64_t mask_nb1; int mask_len;             // mask_len: rows past it are out
    float * weights; int64_t w_nb1, w_nb2;
    char * dst; int64_t d_nb1, d_nb2; int dst_f32;
    float scale_log2;             // scale * log2(e)
    float cap_in, cap_out;        // soft cap c: scale / c and c * log2(e); cap_out = 0: none
    int window, n_seq, n_head, n_head_kv, group, row_blocks, head_blocks, dv, quad;
    int rows;                     // heads of a head block, as partial results lie: row_blocks of up to 16 or 32 (128) a KV head, or (quad) four KV heads' groups
    int n_wg;
    float *  part_o;              // [2 * n_wg][rows][dv]
    float2 * part_ml;             // [2 * n_wg][rows]: maximum (log2 units), sum
    int2 *   items;               // [n_seq * head_blocks]: (2 * first workgroup + whether the item begins inside its run, last workgroup)
    float *  scores;              // [n_seq][n_head][cap] in log2 units, or nullptr
    float2 * lse;                 // [n_seq][n_head]: maximum, 1 / sum
    int64_t  cap;                 // bt_stride * 128
};

// Workgroups a CU holds: a wave's tile of K and V, its Q fragments and its accumulators take up to 256 registers for heads up to 192 wide
// and one block of 16 query heads, more (two waves a SIMD would spill) beyond.
constexpr int wg_per_cu(int dk, int nb) { return dk <= 64 || (dk <= 192 && nb == 1) ? 2 : 1; }

template <bool F16> __device__ __forceinline__ f32x4 mfma16(u32x4 a, u32x4 b, f32x4 c) {
    if constexpr (F16) return __builtin_amdgcn_mfma_f32_16x16x32_f16(bitcast<f16x8>(a), bitcast<f16x8>(b), c, 0, 0, 0);
    else               return __builtin_amdgcn_mfma_f32_16x16x32_bf16(bitcast<bf16x8>(a), bitcast<bf16x8>(b), c, 0, 0, 0);
}
// Values that are the same in every lane, told to the compiler; and lengths and page ids read through the scalar cache (nothing writes them while the
// kernel runs): a vector load among those of K and V would have the wave wait for all that were issued before it.
__device__ __forceinline__ int uni(int v) { return __builtin_amdgcn_readfirstlane(v); }
__device__ __forceinline__ int scalar_at(const int32_t * p, int64_t i) { return *(const int32_t __attribute__((address_space(4))) *) (uintptr_t) (p + i); }

// The rows a sequence attends to, [first, last).
struct Span { int first, last; };
__device__ __forceinline__ Span span_from(const AttnP & p, int n) {
    n = min(max(n, 0), (int) p.cap);                              // (the host has checked that the room is below 2^31)
    const int first = p.window > 0 ? max(n - p.window, 0) : 0;
    n = min(n, p.mask_len);
    return n > first ? Span{ first, n } : Span{ 0, 0 };
}
__device__ __forceinline__ Span span_of(const AttnP & p, int b) { return span_from(p, p.seq_lens[b]); }
__device__ __forceinline__ Span span_uni(const AttnP & p, int b) {        // b the same in every lane
    const Span s = span_from(p, scalar_at(p.seq_lens, b));
    return Span{ uni(s.first), uni(s.last) };
}
__device__ __forceinline__ int pages_of(Span s) { return s.last > s.first ? (s.last + PAGE - 1) / PAGE - s.first / PAGE : 0; }

// Run of workgroup v of n when `total` units are dealt: the first total % n take one more.
struct Deal { int base, more; };
__device__ __forceinline__ int run_start(Deal d, int v) { return v * d.base + min(v, d.more); }
__device__ __forceinline__ int owner_of(Deal d, int unit) {
    const int lead = d.more * (d.base + 1);
    return unit < lead ? unit / (d.base + 1) : d.more + (unit - lead) / d.base;
}

template <int DV> struct VGeom {
    static constexpr int W      = DV >= 128 ? 8 : 4;    // consecutive columns of a lane
    static constexpr int GROUPS = DV / (16 * W);        // such runs, 16 * W columns apart
    static constexpr int COLS   = W * GROUPS;           // MFMAs (columns of a lane)
};

// The deal, computed by every wave for itself (no barrier, and for up to 256 sequences one load of the lengths): how many pages there are, in all
// head blocks, and the sequence of unit u, where a unit is `per` pages of a head block (the last of a head block fewer).  A lane takes 4
// consecutive sequences of 256.
struct Place { int seq, before; };           // the sequence a unit lies in (-1: past the last), and the units before that sequence
struct Lengths {
    int own[4];                              // pages of this lane's sequences
    __device__ __forceinline__ void fetch(const AttnP & p, int lane, int b0) {
#pragma unroll
        for (int e = 0; e < 4; e++) { const int b = b0 + lane * 4 + e; own[e] = b < p.n_seq ? pages_of(span_of(p, b)) : 0; }
    }
    __device__ __forceinline__ int all_pages(const AttnP & p, int lane) {
        int total = 0;
        for (int b0 = 0; b0 < p.n_seq; b0 += 256) { fetch(p, lane, b0); total += lane_of(scan_wave(own[0] + own[1] + own[2] + own[3]), 63); }
        return total * p.head_blocks;
    }
    __device__ __forceinline__ int all_units(const AttnP & p, int lane, int per) {           // after all_pages
        int total = 0;
        for (int b0 = 0; b0 < p.n_seq; b0 += 256) {
            if (p.n_seq > 256) fetch(p, lane, b0);
            int n = 0;
#pragma unroll
            for (int e = 0; e < 4; e++) n += (own[e] + per - 1) / per;
            total += lane_of(scan_wave(n), 63);
        }
        return total * p.head_blocks;
    }
    __device__ __forceinline__ Place place(const AttnP & p, int lane, int u, int per) {      // after all_pages
        for (int b0 = 0, before = 0; b0 < p.n_seq; b0 += 256) {
            if (p.n_seq > 256) fetch(p, lane, b0);
            int n[4];
#pragma unroll
            for (int e = 0; e < 4; e++) n[e] = (per == 1 ? own[e] : (own[e] + per - 1) / per) * p.head_blocks;
            const int mine = n[0] + n[1] + n[2] + n[3], incl = scan_wave(mine), all = lane_of(incl, 63);
            if (u < before + all) {
                const int at = __ffsll(__ballot(u < before + incl)) - 1;      // the first lane whose sequences reach past u
                int ahead = before + lane_of(incl - mine, at), e = 0;
                for (; e < 3; e++) {
                    const int k = lane_of(e == 0 ? n[0] : e == 1 ? n[1] : n[2], at);
                    if (u < ahead + k) break;
                    ahead += k;
                }
                return Place{ b0 + at * 4 + e, ahead };
            }
            before += all;
        }
        return Place{ -1, 0 };
    }
};

// The mask's four numbers of rows t .. t + 3, in one load where their place allows it; rows outside the span: -inf.
__device__ __forceinline__ u32x2 mask4(const AttnP & p, int b, int t, Span s) {
    const char * src = p.mask + (int64_t) b * p.mask_nb1 + (int64_t) t * 2;
    if (t >= s.first && t + 4 <= s.last && ((uintptr_t) src & 7) == 0) return *(const u32x2 *) src;
    unsigned short h[4];
#pragma unroll
    for (int j = 0; j < 4; j++) h[j] = t + j >= s.first && t + j < s.last ? *(const unsigned short *) (src + 2 * j) : (unsigned short) 0xfc00;
    return u32x2{ h[0] | ((unsigned) h[1] << 16), h[2] | ((unsigned) h[3] << 16) };
}
// A score in log2 units from the product q . k, before the mask.  A soft cap c turns a score s into c tanh(y), y = s / c: 1 - 2 / (e^2y + 1) from y = 3/4 on,
// of which a small y would keep no digits; there s itself times tanh(y) / y, by Lambert's continued fraction to y^2 / 9 (off by y^10 / 10^7: 6e-9), so that a
// cap far above the scores leaves them as they are.  Either is off by 2^-21 of itself at most, and they share the reciprocal.
template <bool BIAS> __device__ __forceinline__ float scaled(const AttnP & p, float a) {
    const float s = p.scale_log2 * a;
    if (BIAS && p.cap_out != 0.f) {
        const float y = fabsf(p.cap_in * a), u = y * y;
        const bool  small = y < 0.75f;
        const float r = __builtin_amdgcn_rcpf(small ? fmaf(u, fmaf(u, 15.f, 420.f), 945.f) : fast_exp2(2.f * LOG2E * y) + 1.f);
        return small ? s * (fmaf(u, u + 105.f, 945.f) * r) : copysignf(p.cap_out * fmaf(-2.f, r, 1.f), s);
    }
    return s;
}
// Page `page` of a pool, at a head's offset (products of 32 bits are the scalar unit's; one of 64 would put the address into vector registers).
__device__ __forceinline__ const char * page_base(const char * data, int page, unsigned nb_page, int64_t head) {
    return data + head + (int64_t) ((uint64_t) __umulhi((unsigned) page, nb_page) << 32 | (unsigned) page * nb_page);
}

// Wave w takes quarter w of every page of the run.  QUAD: wave w takes whole pages of KV head w of four, which are the run's head block: a row's four
// heads are read side by side, and the waves have nothing to join.
template <bool F16, int DK, int DV, int NB, bool BIAS, bool QUAD>
__global__ void __launch_bounds__(256, wg_per_cu(DK, NB)) gqa_attn_kernel(const AttnP p) {
    static_assert(NB == 1 || !QUAD, "one block of heads a wave");
    constexpr int  KC    = DK / 32;
    constexpr int  ROWS  = NB * 16, NW = 4;
    // P is taken relative to a reference that lies REF below the maximum when it is set and stays until a score passes that maximum by SLACK (log2 units).
    // Three parts of bf16 hold P to 2^-24 of itself, two of f16 to 2^-22; f16's end at 2^-25, so there P runs up to 2^15, and what is lost of a row is 2^-36 of the largest.
    constexpr int   PARTS = F16 ? 2 : 3;
    constexpr float REF = F16 ? 11.f : 0.f, SLACK = F16 ? 4.f : 8.f;
    using VG = VGeom<DV>;
    extern __shared__ __attribute__((aligned(16))) char lds[];
    __shared__ float2 sh_ml[QUAD ? 1 : NW][ROWS];

    const int lane = threadIdx.x & 63, wave = uni(threadIdx.x >> 6), l15 = lane & 15, lg = lane >> 4;
    const int wg = blockIdx.x;

    // ---- which units are this workgroup's
    Lengths    lens;
    const int  total = lens.all_pages(p, lane);
    const Deal deal{ uni(total / p.n_wg), uni(total % p.n_wg) };
    int        u = uni(run_start(deal, wg));
    const int  u_end = uni(run_start(deal, wg + 1));
    if (u >= u_end) return;
    const Place at = lens.place(p, lane, u, 1);
    int  b = uni(at.seq);
    Span s = span_uni(p, b);
    int  np = uni(pages_of(s));
    int  hb = uni((u - uni(at.before)) / np), pg = u - uni(at.before) - hb * np;

    for (bool fresh = true; u < u_end; fresh = false) {
        b = uni(b); hb = uni(hb); pg = uni(pg); np = uni(np); s = Span{ uni(s.first), uni(s.last) };
        const int  n = uni(min(np - pg, u_end - u));         // pages of this piece
        const bool begins = pg == 0, whole = begins && n == np;
        const int  kvh = QUAD ? hb * 4 + wave : uni(hb / p.row_blocks), row0 = QUAD ? 0 : (hb - kvh * p.row_blocks) * ROWS;   // first head of the group taken here
        const int  heads = min(ROWS, p.group - row0);
        const int  head0 = kvh * p.group + row0;
        if (begins && threadIdx.x == 0) p.items[(int64_t) b * p.head_blocks + hb] = make_int2(2 * wg + (fresh ? 0 : 1), owner_of(deal, u + np - 1));

        const int       bt0 = b * (int) p.bt_stride + s.first / PAGE + pg;       // (the host has checked that it fits)
        const int       t_page0 = (s.first / PAGE + pg) * PAGE;
        u32x4 kf[2][KC];
        u32x2 vf[8][VG::COLS / 4];
        // tile i of this wave: its page of the piece and its first row there
        auto page_of = [&](int i) { return QUAD ? i >> 2 : i; };
        auto slot0 = [&](int i) { return QUAD ? (i & 3) * 32 : wave * 32; };
        // (of four quarters those that have rows)
        const int i_begin = QUAD ? max(s.first - t_page0, 0) / 32 : 0, i_end = QUAD ? min(4 * n, (s.last - t_page0 + 31) / 32) : n;
        // the slots in the page whose rows a lane loads: rows outside the span are replaced by the nearest one inside
        auto slot = [&](int i, int r) { const int t = t_page0 + page_of(i) * PAGE; return min(max(slot0(i) + r, s.first - t), s.last - 1 - t); };
        const int64_t k_off = (int64_t) kvh * p.k_head, v_off = (int64_t) kvh * p.v_head;
        auto load_k = [&](int i, int page) {
            const char * base = page_base(p.k, page, p.k_page, k_off);
#pragma unroll
            for (int blk = 0; blk < 2; blk++) {
                const unsigned row = slot(i, blk * 16 + l15) * p.k_row + lg * 16;
#pragma unroll
                for (int c = 0; c < KC; c++) kf[blk][c] = *(const u32x4 *) (base + row + c * 64);
            }
        };
        auto load_v = [&](int i, int page) {
            const char * base = page_base(p.v, page, p.v_page, v_off);
#pragma unroll
            for (int e = 0; e < 8; e++) {
                const unsigned row = slot(i, (e >> 2) * 16 + lg * 4 + (e & 3)) * p.v_row + l15 * (VG::W * 2);
#pragma unroll
                for (int gr = 0; gr < VG::GROUPS; gr++) {
                    if constexpr (VG::W == 8) {
                        const u32x4 x = *(const u32x4 *) (base + row + gr * 256);
                        vf[e][2 * gr] = u32x2{ x[0], x[1] }; vf[e][2 * gr + 1] = u32x2{ x[2], x[3] };
                    } else vf[e][gr] = *(const u32x2 *) (base + row);
                }
            }
        };
        auto id_at = [&](int i) { return scalar_at(p.block_table, bt0 + min(page_of(i), n - 1)); };        // page id of tile i
        auto good = [&](int id) { return id >= 0 && id < p.n_pages; };          // (a bad id: page 0 is read, not used)

        u32x2 mk[2];                                            // the mask of a tile's rows
        auto load_mask = [&](int i) {
            if constexpr (BIAS)
                if (p.mask)
#pragma unroll
                    for (int blk = 0; blk < 2; blk++) mk[blk] = mask4(p, b, t_page0 + page_of(i) * PAGE + slot0(i) + blk * 16 + lg * 4, s);
        };

        int id = id_at(i_begin), id_next = id_at(i_begin + 1);  // (ids are fetched a tile ahead of their rows)
        load_k(i_begin, good(id) ? id : 0);
        load_v(i_begin, good(id) ? id : 0);
        load_mask(i_begin);
        // ---- Q: operand fragments, lane (h, g) k = 32 c + 8 g .. + 7; heads past the group: zeros
        u32x4 qf[NB * KC];
        auto q_at = [&](int row, int off) { return p.q + (int64_t) b * p.q_nb2 + (int64_t) (head0 + min(row, heads - 1)) * p.q_nb1 + off * (p.q_f32 ? 4 : 2); };   // 8 values from `off` on
        auto q_half = [&](int row, int off) {
            const u32x4 x = *(const u32x4 *) q_at(row, off);
            return row < heads ? x : u32x4{ 0u, 0u, 0u, 0u };
        };
        auto q_full = [&](int row, int off) {
            const f32x4 x = *(const f32x4 *) q_at(row, off), y = *(const f32x4 *) (q_at(row, off) + 16);
            return row < heads ? u32x4{ pair16<F16>(x.x, x.y), pair16<F16>(x.z, x.w), pair16<F16>(y.x, y.y), pair16<F16>(y.z, y.w) } : u32x4{ 0u, 0u, 0u, 0u };
        };
        if (p.q_f32) {
#pragma unroll
            for (int nb = 0; nb < NB; nb++)
#pragma unroll
                for (int c = 0; c < KC; c++) qf[nb * KC + c] = q_full(nb * 16 + l15, c * 32 + lg * 8);
        } else {
#pragma unroll
            for (int nb = 0; nb < NB; nb++)
#pragma unroll
                for (int c = 0; c < KC; c++) qf[nb * KC + c] = q_half(nb * 16 + l15, c * 32 + lg * 8);
        }

        float m[NB], l[NB];
        f32x4 acc[NB][VG::COLS];
#pragma unroll
        for (int nb = 0; nb < NB; nb++) {
            m[nb] = -INFINITY; l[nb] = 0.f;
#pragma unroll
            for (int c = 0; c < VG::COLS; c++) acc[nb][c] = f32x4{ 0.f, 0.f, 0.f, 0.f };
        }

        // One tile; MORE: another one follows (known to the compiler, so that the loads under way are counted: a branch around them would have every
        // wait be for all of them)
        auto tile = [&](auto more_tag, int i) __attribute__((always_inline)) {
            constexpr bool MORE = decltype(more_tag)::value;
            const int  t0 = t_page0 + page_of(i) * PAGE + slot0(i);  // first row of the tile
            const int  lo = max(s.first - t0, 0), hi = min(s.last - t0, 32);
            const bool use = good(id) && hi > lo, all = lo == 0 && hi == 32;
            const int  next = good(id_next) ? id_next : 0;
            id = id_next;
            id_next = id_at(i + 2);

            // the mask's numbers, and the rows it takes out (rows outside the span among them: they repeat one inside, which may be masked)
            float mf[2][4];
            bool  out[2][4];
            if constexpr (BIAS) {
                if (p.mask) {
#pragma unroll
                    for (int blk = 0; blk < 2; blk++)
#pragma unroll
                        for (int j = 0; j < 4; j++) {
                            const float f = f16_bits_to_f32((mk[blk][j >> 1] >> (16 * (j & 1))) & 0xffffu);
                            out[blk][j] = f == -INFINITY;
                            mf[blk][j]  = f * LOG2E;
                        }
                    if constexpr (MORE) load_mask(i + 1);
                }
            }

            u32x4 pf[NB][PARTS];
#pragma unroll
            for (int nb = 0; nb < NB; nb++) {
                f32x4 sc[2] = { { 0.f, 0.f, 0.f, 0.f }, { 0.f, 0.f, 0.f, 0.f } };
#pragma unroll
                for (int c = 0; c < KC; c++) {
                    sc[0] = mfma16<F16>(kf[0][c], qf[nb * KC + c], sc[0]);
                    sc[1] = mfma16<F16>(kf[1][c], qf[nb * KC + c], sc[1]);
                }
                if (MORE && nb == NB - 1) load_k(i + 1, next);

                float x[8];                                     // scores in log2 units
#pragma unroll
                for (int e = 0; e < 8; e++) {
                    x[e] = scaled<BIAS>(p, sc[e >> 2][e & 3]);
                    if constexpr (BIAS) if (p.mask) x[e] = out[e >> 2][e & 3] ? -INFINITY : x[e] + mf[e >> 2][e & 3];
                }
                if (!use || !all) {
#pragma unroll
                    for (int e = 0; e < 8; e++) {
                        const int r = (e >> 2) * 16 + lg * 4 + (e & 3);
                        if (!use || r < lo || r >= hi) x[e] = -INFINITY;
                    }
                }
                if (p.scores && nb * 16 + l15 < heads) {
                    float * to = p.scores + ((int64_t) b * p.n_head + head0 + nb * 16 + l15) * p.cap + t0 + lg * 4;
                    *(f32x4 *) to        = f32x4{ x[0], x[1], x[2], x[3] };
                    *(f32x4 *) (to + 16) = f32x4{ x[4], x[5], x[6], x[7] };
                }
                float top = x[0];
#pragma unroll
                for (int e = 1; e < 8; e++) top = fmaxf(top, x[e]);
                if (__any(top > m[nb] + (REF + SLACK))) {
                    top = fmaxf(top, __shfl_xor(top, 16, 64));
                    top = fmaxf(top, __shfl_xor(top, 32, 64));
                    const float nm = fmaxf(top - REF, m[nb]);
                    const float a  = m[nb] == nm ? 1.f : fast_exp2(m[nb] - nm);
                    m[nb] = nm;
                    l[nb] *= a;
#pragma unroll
                    for (int j = 0; j < 4; j++) {
                        const float aj = __shfl(a, lg * 4 + j, 64);
#pragma unroll
                        for (int c = 0; c < VG::COLS; c++) acc[nb][c][j] *= aj;
                    }
                }
                const float mm = m[nb] == -INFINITY ? 0.f : m[nb];
#pragma unroll
                for (int e = 0; e < 8; e++) { x[e] = fast_exp2(x[e] - mm); l[nb] += x[e]; }
#pragma unroll
                for (int e = 0; e < 4; e++)
#pragma unroll
                    for (int part = 0; part < PARTS; part++) {  // what is left of it each time (exact)
                        const unsigned h = pf[nb][part][e] = pair16<F16>(x[2 * e], x[2 * e + 1]);
                        x[2 * e]     -= from16<F16>((unsigned short) h);
                        x[2 * e + 1] -= from16<F16>((unsigned short) (h >> 16));
                    }
            }
            if (use) {
                if constexpr (BIAS) {
                    // a row the mask takes out has p = 0, and 0 * NaN must not count
                    if (p.mask) {
#pragma unroll
                        for (int e = 0; e < 8; e++)
#pragma unroll
                            for (int c = 0; c < VG::COLS / 4; c++)
                                if (out[e >> 2][e & 3]) vf[e][c] = u32x2{ 0u, 0u };
                    }
                }
#pragma unroll
                for (int c = 0; c < VG::COLS; c++) {
                    u32x4 bf;
#pragma unroll
                    for (int e = 0; e < 4; e++)
                        bf[e] = __builtin_amdgcn_perm(vf[2 * e + 1][c >> 2][(c >> 1) & 1], vf[2 * e][c >> 2][(c >> 1) & 1], c & 1 ? 0x07060302u : 0x05040100u);
#pragma unroll
                    for (int nb = 0; nb < NB; nb++)
#pragma unroll
                        for (int part = 0; part < PARTS; part++) acc[nb][c] = mfma16<F16>(pf[nb][part], bf, acc[nb][c]);
                }
            }
            if constexpr (MORE) load_v(i + 1, next);
        };
        int i = i_begin;
        for (; i + 1 < i_end; i++) tile(std::true_type{}, i);
        tile(std::false_type{}, i);

        const int64_t piece = 2 * (int64_t) wg + (fresh ? 0 : 1);
#pragma unroll
        for (int nb = 0; nb < NB; nb++) {
            l[nb] += __shfl_xor(l[nb], 16, 64);
            l[nb] += __shfl_xor(l[nb], 32, 64);
        }
        if constexpr (QUAD) {
            const float inv = l[0] == 0.f ? 0.f : 1.f / l[0];    // (a NaN stays one)
            if (lg == 0 && l15 < heads) {
                if (!whole) p.part_ml[piece * p.rows + wave * p.group + l15] = make_float2(m[0], l[0]);
                else if (p.scores) p.lse[(int64_t) b * p.n_head + head0 + l15] = make_float2(m[0] == -INFINITY ? 0.f : m[0], inv);
            }
#pragma unroll
            for (int j = 0; j < 4; j++) {
                const int   row = lg * 4 + j;
                const float f = whole ? __shfl(inv, row, 64) : 1.f;
                if (row >= heads) continue;
                char *  dst = p.dst + (int64_t) b * p.d_nb2 + (int64_t) (head0 + row) * p.d_nb1;
                float * part = p.part_o + (piece * p.rows + wave * p.group + row) * DV;
#pragma unroll
                for (int gr = 0; gr < VG::GROUPS; gr++)
#pragma unroll
                    for (int c = 0; c < VG::W; c += 4) {
                        const int   a = gr * VG::W + c, col = gr * 128 + l15 * VG::W + c;
                        const f32x4 o = f32x4{ acc[0][a][j], acc[0][a + 1][j], acc[0][a + 2][j], acc[0][a + 3][j] } * f;
                        if (!whole)         *(f32x4 *) (part + col) = o;
                        else if (p.dst_f32) *(f32x4 *) (dst + col * 4) = o;
                        else                *(u32x2 *) (dst + col * 2) = u32x2{ pair16<F16>(o.x, o.y), pair16<F16>(o.z, o.w) };
                    }
            }
        } else {
        // ---- the waves' results meet in LDS
#pragma unroll
        for (int nb = 0; nb < NB; nb++)
            if (lg == 0) sh_ml[wave][nb * 16 + l15] = make_float2(m[nb], l[nb]);
        __syncthreads();
        auto joined = [&](int row) -> float2 {               // maximum and sum over the waves
            float M = -INFINITY, L = 0.f;
#pragma unroll
            for (int w = 0; w < NW; w++) M = fmaxf(M, sh_ml[w][row].x);
#pragma unroll
            for (int w = 0; w < NW; w++) L += sh_ml[w][row].y == 0.f ? 0.f : sh_ml[w][row].y * fast_exp2(sh_ml[w][row].x - M);
            return make_float2(M, L);
        };
        for (int r = threadIdx.x; r < heads; r += 256) {
            const float2 ml = joined(r);
            if (!whole) p.part_ml[piece * p.rows + r] = ml;
            else if (p.scores) p.lse[(int64_t) b * p.n_head + head0 + r] = make_float2(ml.x == -INFINITY ? 0.f : ml.x, ml.y == 0.f ? 0.f : 1.f / ml.y);
        }
        float * part = (float *) lds;                         // [4][16][DV]
#pragma unroll
        for (int nb = 0; nb < NB; nb++) {
            if (nb) __syncthreads();
#pragma unroll
            for (int j = 0; j < 4; j++) {
                const int    row = nb * 16 + lg * 4 + j;
                const float  mw  = sh_ml[wave][row].x;
                const float2 ml  = joined(row);
                const float  f   = mw == -INFINITY ? 0.f : fast_exp2(mw - ml.x);
                float * to = part + (wave * 16 + lg * 4 + j) * DV + l15 * VG::W;
#pragma unroll
                for (int gr = 0; gr < VG::GROUPS; gr++)
#pragma unroll
                    for (int c = 0; c < VG::W; c += 4) {
                        const int a = gr * VG::W + c;
                        *(f32x4 *) (to + gr * 128 + c) = f32x4{ acc[nb][a][j] * f, acc[nb][a + 1][j] * f, acc[nb][a + 2][j] * f, acc[nb][a + 3][j] * f };
                    }
            }
            __syncthreads();
            for (int i = threadIdx.x; i < 4 * DV; i += 256) {     // 16 rows of DV / 4 runs of 4
                const int r = i / (DV / 4), c = (i - r * (DV / 4)) * 4, row = nb * 16 + r;
                if (row >= heads) continue;
                f32x4 o = *(const f32x4 *) (part + r * DV + c);
#pragma unroll
                for (int w = 1; w < 4; w++) o += *(const f32x4 *) (part + (w * 16 + r) * DV + c);
                if (!whole) *(f32x4 *) (p.part_o + (piece * p.rows + row) * DV + c) = o;
                else {
                    const float L = joined(row).y, inv = L == 0.f ? 0.f : 1.f / L;   // (a NaN stays one)
                    char * to = p.dst + (int64_t) b * p.d_nb2 + (int64_t) (head0 + row) * p.d_nb1;
                    o *= inv;
                    if (p.dst_f32) *(f32x4 *) (to + c * 4) = o;
                    else *(u32x2 *) (to + c * 2) = u32x2{ pair16<F16>(o.x, o.y), pair16<F16>(o.z, o.w) };
                }
            }
        }
        __syncthreads();                                      // LDS is free again for the next piece
        }

        u += n; pg = 0;
        if (++hb == p.head_blocks && u < u_end) {
            hb = 0;
            do { b++; s = span_uni(p, b); np = uni(pages_of(s)); } while (np == 0);   // (u < u_end <= total: there is such a sequence)
        }
    }
}

// Scores of a latent cache (rows of 576, one KV head) for its weights: (m, l) and every score, as gqa_attn_kernel leaves them, without V.  Up to
// 128 heads share a row, 128 flop a byte: the rows of Q lie in LDS (147 KB) and are read, 16 heads at a time, against a tile of 32 rows of K
// in registers, by eight waves, so that every SIMD still has two.  The loop over blocks of heads is a loop: eight copies of its body, run once or
// twice by a workgroup, took twice as long, most of it to fetch them.  8 x 8192 rows, 128 heads: 30 us (8 of 5000
// to 8192 rows: 27), of which the rows are 12 at the memory's rate, the products 4 to 7 and the reads of Q from LDS 4 side by side: what bounds it is one tile a
// wave behind the staging of Q, and a chain of LDS reads, products, shuffles and exp2 a block of heads; then 4 to join and 8 to add them up.
constexpr int LK = 576, LPITCH = LK * 2 + 16, LWAVES = 8, LROWS = 128;
template <bool F16, bool BIAS>
__global__ void __launch_bounds__(64 * LWAVES) gqa_scores_kernel(const AttnP p) {
    constexpr int KC = LK / 32;
    extern __shared__ __attribute__((aligned(16))) char lds[];
    __shared__ float2 sh_ml[LWAVES][LROWS];
    const int lane = threadIdx.x & 63, wave = uni(threadIdx.x >> 6), quarter = wave & 3, l15 = lane & 15, lg = lane >> 4;
    const int wg = blockIdx.x;
    // A workgroup's Q is 147 KB to stage, so no run crosses from one (sequence, head block) to another: units of `per` pages, the fewest of which
    // there are no more than workgroups (units of `top` pages are never more; taking those, 8 x 8192 rows came to 3 pages a unit and 37 us, not 2 and 30); with as many head blocks as workgroups, whole ones in turn.
    Lengths   lens;
    const int total = lens.all_pages(p, lane), spare = p.n_wg - p.n_seq * p.head_blocks;
    int per = INT_MAX / 2;
    if (spare > 0) {
        per = uni((total + p.n_wg - 1) / p.n_wg);
        for (int top = uni((total + spare - 1) / spare); per < top;) {
            const int mid = (per + top) / 2;
            if (uni(lens.all_units(p, lane, max(mid, 1))) <= p.n_wg) top = mid;
            else per = mid + 1;
        }
        per = max(per, 1);
    }
    for (int u = wg;; u += p.n_wg) {
        const Place at = lens.place(p, lane, u, per);
        const int b = uni(at.seq);
        if (b < 0) return;
        const Span s = span_uni(p, b);
        const int np = uni(pages_of(s)), units = uni((np + per - 1) / per);
        const int hb = uni((u - uni(at.before)) / units), pg = (u - uni(at.before) - hb * units) * per;
        const int n = uni(min(np - pg, per));
        const bool whole = n == np;
        const int  head0 = hb * LROWS, heads = min(LROWS, p.group - head0);
        if (pg == 0 && threadIdx.x == 0) p.items[(int64_t) b * p.head_blocks + hb] = make_int2(2 * u, u + units - 1);    // (units of one: u < n_wg)
        const int bt0 = b * (int) p.bt_stride + s.first / PAGE + pg, t_page0 = (s.first / PAGE + pg) * PAGE;
        auto id_at = [&](int i) { return scalar_at(p.block_table, bt0 + min(i, n - 1)); };
        auto good = [&](int id) { return id >= 0 && id < p.n_pages; };
        u32x4 kf[2][KC];
        auto load_k = [&](int i, int page) {
            const char * base = page_base(p.k, page, p.k_page, 0);
#pragma unroll
            for (int blk = 0; blk < 2; blk++) {
                const int t = t_page0 + i * PAGE;
                const unsigned row = min(max(quarter * 32 + blk * 16 + l15, s.first - t), s.last - 1 - t) * p.k_row + lg * 16;
#pragma unroll
                for (int c = 0; c < KC; c++) kf[blk][c] = *(const u32x4 *) (base + row + c * 64);
            }
        };
        int i = wave >> 2;                                     // waves 0 .. 3 the even pages of the unit, 4 .. 7 the odd ones
        int id = id_at(i);

        // ---- Q to LDS, six pieces a thread under way at a time, the first tile of K behind the last six; rows past the group: zeros
        constexpr int PIECES = LROWS * (LK / 8) / (64 * LWAVES);
        static_assert(PIECES * 64 * LWAVES == LROWS * (LK / 8) && PIECES % 6 == 0, "whole pieces");
        auto stage = [&](int k0, auto behind) {
            u32x4 v[6], w[6];
            auto row_of = [&](int k) { return (int) (threadIdx.x + (k0 + k) * 64 * LWAVES) / (LK / 8); };
            auto col_of = [&](int k) { return (int) (threadIdx.x + (k0 + k) * 64 * LWAVES) % (LK / 8); };
            auto src = [&](int k) { return p.q + (int64_t) b * p.q_nb2 + (int64_t) (head0 + min(row_of(k), heads - 1)) * p.q_nb1 + col_of(k) * (p.q_f32 ? 32 : 16); };
#pragma unroll
            for (int k = 0; k < 6; k++) v[k] = *(const u32x4 *) src(k);
            if (p.q_f32) {
#pragma unroll
                for (int k = 0; k < 6; k++) w[k] = *(const u32x4 *) (src(k) + 16);
#pragma unroll
                for (int k = 0; k < 6; k++) {
                    const f32x4 x = bitcast<f32x4>(v[k]), y = bitcast<f32x4>(w[k]);
                    v[k] = u32x4{ pair16<F16>(x.x, x.y), pair16<F16>(x.z, x.w), pair16<F16>(y.x, y.y), pair16<F16>(y.z, y.w) };
                }
            }
            behind();
            __builtin_amdgcn_sched_barrier(0);
#pragma unroll
            for (int k = 0; k < 6; k++) *(u32x4 *) (lds + row_of(k) * LPITCH + col_of(k) * 16) = row_of(k) < heads ? v[k] : u32x4{ 0u, 0u, 0u, 0u };
        };
        const int last = uni((min(LROWS, (heads + 15) & ~15) * (LK / 8) - 1) / (6 * 64 * LWAVES)) * 6;    // (blocks of 16 rows without a head are not read)
#pragma unroll 1
        for (int k0 = 0; k0 < last; k0 += 6) stage(k0, [] {});
        stage(last, [&] { load_k(min(i, n - 1), good(id) ? id : 0); });           // (a wave without a page of its own: the last one's, unused)
        // (a wave's own rows of sh_ml hold its running maxima and sums; what lanes 0 .. 15 write of a page the others read with the next one: a fence between)
        for (int r = lane; r < LROWS; r += 64) sh_ml[wave][r] = make_float2(-INFINITY, 0.f);
        __syncthreads();

        for (; i < n; i += LWAVES / 4) {
            const int  t0 = t_page0 + i * PAGE + quarter * 32;
            const bool use = good(id);
            id = id_at(i + LWAVES / 4);
            u32x2 mk[2] = { { 0u, 0u }, { 0u, 0u } };
            if constexpr (BIAS)
                if (p.mask)
#pragma unroll
                    for (int blk = 0; blk < 2; blk++) mk[blk] = mask4(p, b, t0 + blk * 16 + lg * 4, s);
            float * to = p.scores + ((int64_t) b * p.n_head + head0 + l15) * p.cap + t0 + lg * 4;
#pragma unroll 1
            for (int h = l15; h - l15 < heads; h += 16, to += 16 * p.cap) {
                f32x4 sc[2] = { { 0.f, 0.f, 0.f, 0.f }, { 0.f, 0.f, 0.f, 0.f } };
                const char * q = lds + h * LPITCH + lg * 16;
#pragma unroll
                for (int c = 0; c < KC; c++) {
                    const u32x4 qq = *(const u32x4 *) (q + c * 64);
                    sc[0] = mfma16<F16>(kf[0][c], qq, sc[0]);
                    sc[1] = mfma16<F16>(kf[1][c], qq, sc[1]);
                }
                float x[8], top = -INFINITY;
#pragma unroll
                for (int e = 0; e < 8; e++) {
                    const int r = t0 + (e >> 2) * 16 + lg * 4 + (e & 3);
                    x[e] = scaled<BIAS>(p, sc[e >> 2][e & 3]);
                    if constexpr (BIAS)
                        if (p.mask) {
                            const float f = f16_bits_to_f32((mk[e >> 2][(e >> 1) & 1] >> (16 * (e & 1))) & 0xffffu);
                            x[e] = f == -INFINITY ? -INFINITY : x[e] + f * LOG2E;
                        }
                    if (!use || r < s.first || r >= s.last) x[e] = -INFINITY;
                    top = fmaxf(top, x[e]);
                }
                if (h < heads) {
                    *(f32x4 *) to        = f32x4{ x[0], x[1], x[2], x[3] };
                    *(f32x4 *) (to + 16) = f32x4{ x[4], x[5], x[6], x[7] };
                }
                const float2 ml = sh_ml[wave][h];
                top = fmaxf(top, __shfl_xor(top, 16, 64));
                top = fmaxf(fmaxf(top, __shfl_xor(top, 32, 64)), ml.x);
                const float mm = top == -INFINITY ? 0.f : top;
                float l = 0.f;
#pragma unroll
                for (int e = 0; e < 8; e++) l += fast_exp2(x[e] - mm);
                l += __shfl_xor(l, 16, 64);
                l += __shfl_xor(l, 32, 64);
                if (lg == 0) sh_ml[wave][h] = make_float2(top, l + (ml.y == 0.f ? 0.f : ml.y * fast_exp2(ml.x - mm)));
            }
            wave_fence();
            if (i + LWAVES / 4 < n) load_k(i + LWAVES / 4, good(id) ? id : 0);
        }
        __syncthreads();
        const int64_t piece = 2 * (int64_t) u;
        for (int r = threadIdx.x; r < heads; r += 64 * LWAVES) {
            float M = -INFINITY, L = 0.f;
#pragma unroll
            for (int w = 0; w < LWAVES; w++) M = fmaxf(M, sh_ml[w][r].x);
#pragma unroll
            for (int w = 0; w < LWAVES; w++) L += sh_ml[w][r].y == 0.f ? 0.f : sh_ml[w][r].y * fast_exp2(sh_ml[w][r].x - M);
            if (!whole) p.part_ml[piece * p.rows + r] = make_float2(M, L);
            else        p.lse[(int64_t) b * p.n_head + head0 + r] = make_float2(M == -INFINITY ? 0.f : M, L == 0.f ? 0.f : 1.f / L);
        }
        __syncthreads();                                       // LDS is free again for the next unit
    }
}

// Joins what the runs left of one head: o = sum_i o_i 2^(m_i - M) / sum_i l_i 2^(m_i - M), pieces in the order of the rows, eight under
// way at a time a thread.  Heads whose rows one run covered are done; heads without a row get zeros.
constexpr int JOIN = 256;
template <bool F16>
__device__ __forceinline__ void join_head(const AttnP & p, int b, int kvh, int r, f32x4 * sum) {
    __shared__ float  red[2][JOIN / 64], weight[JOIN];
    const int h = kvh * p.group + r;
    const int hb = p.quad ? kvh >> 2 : kvh * p.row_blocks + r / p.rows, row = p.quad ? (kvh & 3) * p.group + r : r % p.rows;
    char *    dst = p.dst + (int64_t) b * p.d_nb2 + (int64_t) h * p.d_nb1;
    const int cols = p.dv / 4;                                // runs of 4 columns
    auto store = [&](int c, f32x4 o) {
        if (p.dst_f32) *(f32x4 *) (dst + c * 16) = o;
        else *(u32x2 *) (dst + c * 8) = u32x2{ pair16<F16>(o.x, o.y), pair16<F16>(o.z, o.w) };
    };
    const int2 it = p.items[(int64_t) b * p.head_blocks + hb];   // (meaningless, and not used, where there is no row)
    if (pages_of(span_of(p, b)) == 0) {
        for (int c = threadIdx.x; c < cols; c += JOIN) store(c, f32x4{ 0.f, 0.f, 0.f, 0.f });
        return;
    }
    const int  v0 = it.x >> 1, n = it.y - v0 + 1;
    if (n == 1) return;
    auto slot = [&](int i) -> int64_t { return ((int64_t) (i ? 2 * (v0 + i) : it.x)) * p.rows + row; };
    auto over_waves = [&](float v, bool maximum) {            // the same in every thread
#pragma unroll
        for (int d = 1; d < 64; d <<= 1) { const float o = __shfl_xor(v, d, 64); v = maximum ? fmaxf(v, o) : v + o; }
        if ((threadIdx.x & 63) == 0) red[maximum][threadIdx.x >> 6] = v;
        __syncthreads();
        v = red[maximum][0];
        for (int w = 1; w < JOIN / 64; w++) v = maximum ? fmaxf(v, red[maximum][w]) : v + red[maximum][w];
        return v;
    };
    // rows and factors of the first pieces are requested together: after the item's, their addresses depend on nothing
    const int groups = JOIN / cols, g = (int) threadIdx.x / cols, c = (int) threadIdx.x - g * cols;   // (cols: 16, 32 or 64)
    f32x4 x[8];
    auto rows = [&](int k, int end) {                         // pieces k, k + groups, ..; past the end: the last one
#pragma unroll
        for (int e = 0; e < 8; e++) x[e] = *(const f32x4 *) (p.part_o + slot(min(k + e * groups, end - 1)) * p.dv + c * 4);
    };
    const float2 first = (int) threadIdx.x < n ? p.part_ml[slot(threadIdx.x)] : make_float2(-INFINITY, 0.f);
    rows(g, min(JOIN, n));
    float M = first.x;
    for (int i = threadIdx.x + JOIN; i < n; i += JOIN) M = fmaxf(M, p.part_ml[slot(i)].x);
    M = over_waves(M, true);
    // pieces in runs of JOIN: their factors, then their rows
    float L = 0.f;
    f32x4 o = { 0.f, 0.f, 0.f, 0.f };
    for (int i0 = 0; i0 < n; i0 += JOIN) {
        const int    end = min(i0 + JOIN, n);
        const float2 ml  = i0 == 0 ? first : i0 + (int) threadIdx.x < end ? p.part_ml[slot(i0 + threadIdx.x)] : make_float2(0.f, 0.f);
        const float  w   = ml.y == 0.f ? 0.f : fast_exp2(ml.x - M);
        L += ml.y * w;
        if (i0) __syncthreads();
        weight[threadIdx.x] = w;
        __syncthreads();
        for (int k = i0 + g; k < end; k += groups * 8) {
            if (k >= groups) rows(k, end);                    // (the first ones are here)
#pragma unroll
            for (int e = 0; e < 8; e++) if (k + e * groups < end) o += x[e] * weight[k + e * groups - i0];
        }
    }
    L = over_waves(L, false);
    const float inv = L == 0.f ? 0.f : 1.f / L;
    if (p.scores && threadIdx.x == 0) p.lse[(int64_t) b * p.n_head + h] = make_float2(M == -INFINITY ? 0.f : M, inv);
    sum[threadIdx.x] = o;
    __syncthreads();
    if (g == 0) {
        for (int i = 1; i < groups; i++) o += sum[i * cols + c];
        store(c, o * inv);
    }
}

// (m, 1 / l) of head r of a group from its pieces, by `lanes` lanes of a wave (a power of two), this one `sub`; all of them get it.  AHEAD pieces a
// lane are under way at a time, and what `meanwhile` requests behind the first.
template <int AHEAD, typename F>
__device__ __forceinline__ float2 join_sums(const AttnP & p, int b, int kvh, int r, int lanes, int sub, F meanwhile) {
    const int  hb = p.quad ? kvh >> 2 : kvh * p.row_blocks + r / p.rows, row = p.quad ? (kvh & 3) * p.group + r : r % p.rows;
    const int2 it = p.items[(int64_t) b * p.head_blocks + hb];
    const int  v0 = it.x >> 1, n = it.y - v0 + 1, slot0 = n > 1 ? it.x : 0;     // (a head of one run left no piece: the first of all is read, unused)
    const float2 whole = p.lse[(int64_t) b * p.n_head + kvh * p.group + r];     // (of a head that one run covered; else meaningless)
    float2 ml[AHEAD];
    auto pieces = [&](int i0) {
#pragma unroll
        for (int e = 0; e < AHEAD; e++) {
            const int i = min(i0 + e * lanes, n - 1);
            ml[e] = p.part_ml[((int64_t) (i ? 2 * (v0 + i) : slot0)) * p.rows + row];
        }
    };
    pieces(sub);
    meanwhile();
    if (n == 1) return whole;
    float M = -INFINITY, L = 0.f;
    for (int i0 = sub; i0 < n; i0 += AHEAD * lanes) {
        if (i0 != sub) pieces(i0);
        float top = M;
#pragma unroll
        for (int e = 0; e < AHEAD; e++) top = fmaxf(top, ml[e].x);
        L = L == 0.f ? 0.f : L * fast_exp2(M - top);
#pragma unroll
        for (int e = 0; e < AHEAD; e++) L += i0 + e * lanes >= n || ml[e].y == 0.f ? 0.f : ml[e].y * fast_exp2(ml[e].x - top);
        M = top;
    }
    for (int d = 1; d < lanes; d <<= 1) {
        const float m = __shfl_xor(M, d, 64), l = __shfl_xor(L, d, 64), top = fmaxf(M, m);
        L = (L == 0.f ? 0.f : L * fast_exp2(M - top)) + (l == 0.f ? 0.f : l * fast_exp2(m - top));
        M = top;
    }
    return make_float2(M == -INFINITY ? 0.f : M, L == 0.f ? 0.f : 1.f / L);
}
// The same for all heads ahead of the sums, a wave a head, where there is no result to join.  Grid: x = the heads of a group in fours, y = a (sequence, KV head).
__global__ void __launch_bounds__(JOIN) gqa_lse_kernel(const AttnP p) {
    const int b = blockIdx.y / p.n_head_kv, kvh = blockIdx.y - b * p.n_head_kv, r = (int) blockIdx.x * 4 + ((int) threadIdx.x >> 6);
    if (r >= p.group || pages_of(span_of(p, b)) == 0) return;
    const float2 got = join_sums<4>(p, b, kvh, r, 64, (int) threadIdx.x & 63, [] {});
    if ((threadIdx.x & 63) == 0) p.lse[(int64_t) b * p.n_head + kvh * p.group + r] = got;
}

// weights[b][g][i] += sum over the group's heads of exp2(s - m) / l, from the scores the first kernel left.  A thread takes 4 rows and
// every parts-th head (parts: 16, or the power of two that holds a smaller group); the parts are added in one order.  (m, l) of a head is
// joined from its pieces by every workgroup for itself, while its first scores are under way, or, ready, by a launch ahead.
constexpr int SUM_HEADS = 256, SUM_BLOCKS = 2048;
template <int HEADS>                                          // scores under way at a time
__device__ __forceinline__ void sum_weights(const AttnP & p, int b, int kvh, int block, int blocks, int parts, bool ready, f32x4 * sum) {
    __shared__ float2 lse[SUM_HEADS];
    const Span s = span_of(p, b);
    const int  quads = JOIN / parts, part = (int) threadIdx.x / quads, quad = (int) threadIdx.x - part * quads, rows = quads * 4;
    const int64_t h0 = (int64_t) b * p.n_head + (int64_t) kvh * p.group;
    auto join = [&](int c, int heads, auto load) {            // heads c .. c + heads - 1 of the group, some lanes of a wave each, and the first scores
        int lanes = 64;
        while (lanes * heads > JOIN) lanes >>= 1;
        const int h = (int) threadIdx.x / lanes, sub = (int) threadIdx.x & (lanes - 1), r = c + min(h, heads - 1);
        float2 got;
        if (ready) { got = p.lse[h0 + r]; load(c + part); }
        else got = join_sums<HEADS == 1 ? 2 : 8>(p, b, kvh, r, lanes, sub, [&] { load(c + part); });      // (16 lanes a head or more, or 1)
        if (h < heads && sub == 0) lse[h] = got;
        __syncthreads();
    };
    bool first = true;
    for (int rb = s.first / rows + block; rb * rows < s.last; rb += blocks, first = false) {
        const int  t  = rb * rows + quad * 4;
        const bool in = t < s.last && t + 4 > s.first;
        f32x4 w = { 0.f, 0.f, 0.f, 0.f };
        for (int c = 0; c < p.group; c += SUM_HEADS) {
            const int end = min(c + SUM_HEADS, p.group);
            f32x4 x[HEADS];
            const float * from = p.scores + h0 * p.cap + (in ? t : s.first & ~3);
            auto load = [&](int h) {                          // heads h, h + parts, ..; past the end: the last one
#pragma unroll
                for (int e = 0; e < HEADS; e++) x[e] = *(const f32x4 *) (from + (int64_t) min(h + e * parts, end - 1) * p.cap);
            };
            if (first || p.group > SUM_HEADS) {
                if (!first || c) __syncthreads();             // (the heads before these are done with)
                join(c, end - c, load);
            } else load(c + part);
            for (int h = c + part; h < end; h += HEADS * parts) {
                if (h >= c + parts) load(h);
#pragma unroll
                for (int e = 0; e < HEADS; e++) {
                    if (h + e * parts >= end) break;
                    const float2 ml = lse[h + e * parts - c];
#pragma unroll
                    for (int j = 0; j < 4; j++) w[j] += fast_exp2(x[e][j] - ml.x) * ml.y;
                }
            }
        }
        if (parts > 1) {
            if (!first) __syncthreads();
            sum[threadIdx.x] = w;
            __syncthreads();
            if (part == 0) for (int q = 1; q < parts; q++) w += sum[q * quads + quad];
        }
        if (part || !in) continue;
        float * to = (float *) ((char *) p.weights + (int64_t) b * p.w_nb2 + (int64_t) kvh * p.w_nb1) + t;
#pragma unroll
        for (int j = 0; j < 4; j++) if (t + j >= s.first && t + j < s.last) to[j] += w[j];
    }
}

// What follows the runs, in one launch.  Grid: x = the heads of a group (none without a result), then the workgroups that share a sequence's
// rows (none without weights); y = a (sequence, KV head).
template <bool F16, int HEADS>
__global__ void __launch_bounds__(JOIN) gqa_join_kernel(const AttnP p, const int joins, const int parts, const int ready) {
    __shared__ f32x4 sum[JOIN];
    const int b = blockIdx.y / p.n_head_kv, kvh = blockIdx.y - b * p.n_head_kv;
    if ((int) blockIdx.x < joins) join_head<F16>(p, b, kvh, (int) blockIdx.x, sum);
    else if constexpr (HEADS > 0) sum_weights<HEADS>(p, b, kvh, (int) blockIdx.x - joins, (int) gridDim.x - joins, parts, ready != 0, sum);
}

// ---------------------------------------------------------------- host

struct Plan {
    int     nb, rows, row_blocks, head_blocks, n_wg;
    bool    quad;
    int64_t items;
    int     pieces;                                           // of a head, where all sequences fill the block table
    size_t  off_ml, off_items, off_scores, off_lse, bytes;    // of the workspace; partial rows first
};

// Both sides of the rules below: whole calls on one MI355X, bf16, pages in brackets (of all KV heads, as many as the block table has room for).
// Two blocks of 16 heads a wave against one: 64 heads on 2 of 128, 64 x 16384 rows (16384) 198 against 316 us, 32 x 8192 (4096) 54 against 90,
// 32 x 2048 (1024) 26 against 32; 32 on 1 of 128, 8 x 16384 (1024) 23.3 against 22.6, 32 x 2048 (512) 20.4 against 18.0, 1 x 1024 14.3 against 11.4.
// Four KV heads a workgroup against one, rows row by row: 16 heads on 16 of 64, 32 x 8192 (32768) 187 against 220, 4 x 4096 (2048) 18.6 against 20.6;
// 16 on 16 of 192 / 128, 8 x 16384 (16384) 228 against 237; 32 on 8 of 128, 8 x 16384 (8192) 101 against 111, 4 x 4096 (1024) 20.3 against 20.1; 16 on 4
// of 64, 32 x 8192 (8192) 51 against 52, 1 x 131072 (4096) 33.3 against 29.5.  Head by head a page of a head is contiguous anyway: 32 on 8 of 128,
// 32 x 8192 194 against 186.  Heads of 256, 512 bytes a row each: 187 against 187.
constexpr int64_t TWO_BLOCKS = 1024, QUADS_OF_MANY = 2048, QUADS = 8192;
// Where weights are summed, heads are joined ahead of the sums if a workgroup of the sums would have this many pieces to read first (pieces of a head, in
// brackets times heads of a group): 128 heads over one latent cache, 1 x 65536 rows (32768) 41 against 65 us, 8 x 8192 (4096) 42 against 42, 8 x 2048
// (2048) 31.5 against 29.5; 16 heads over it, 1 x 65536 (4096) 27 against 31; 32 on 8 of 128, 8 x 2048 (128) 25.1 against 21.2.
constexpr int64_t JOIN_AHEAD = 4096;
Plan make_plan(const gqa_attn_args * a) {
    Plan pl;
    const int group = a->n_head / a->n_head_kv;
    const int64_t pages = (int64_t) a->n_seq * a->n_head_kv * a->bt_stride;      // at most
    // blocks of 16 heads a wave holds: two where the group fills them and the registers allow it (heads of 256: a second block has its own workgroups,
    // which find K and V in the caches), eight over a latent cache, whose Q lies in LDS
    pl.nb = a->dv == 0 ? LROWS / 16 : group > 16 && a->dk < 256 && pages >= TWO_BLOCKS ? 2 : 1;
    // four KV heads a workgroup where a row's heads lie side by side in both caches
    const bool side = a->k.nb_row >= a->n_head_kv * a->k.nb_head && a->v.nb_row >= a->n_head_kv * a->v.nb_head;
    pl.quad = a->dv != 0 && a->dk < 256 && group <= 16 && a->n_head_kv % 4 == 0 && side && pages >= (a->n_head_kv >= 8 ? QUADS_OF_MANY : QUADS);
    pl.rows = pl.quad ? 4 * group : pl.nb * 16;
    pl.row_blocks = pl.quad ? 1 : (group + pl.rows - 1) / pl.rows;
    pl.head_blocks = pl.quad ? a->n_head_kv / 4 : a->n_head_kv * pl.row_blocks;
    pl.items = (int64_t) a->n_seq * pl.head_blocks;
    const int64_t units = pl.items * a->bt_stride + (a->dv ? 0 : pl.items);       // (the scores' deal keeps a workgroup an item aside for what is left over)
    const int fill = 256 * (a->dv ? wg_per_cu(a->dk, pl.nb) : 1);
    pl.n_wg = (int) (units < fill ? units : fill);
    if (a->n_workgroups > 0) pl.n_wg = (int) (units < a->n_workgroups ? units : a->n_workgroups);
    const int64_t shares = (pl.n_wg + pl.items - 1) / pl.items;
    pl.pieces = (int) (shares < a->bt_stride ? shares : a->bt_stride);
    size_t at = 0;
    auto take = [&](size_t n) { const size_t o = at; at += (n + 255) & ~(size_t) 255; return o; };
    take((size_t) 2 * pl.n_wg * pl.rows * a->dv * 4);
    pl.off_ml    = take((size_t) 2 * pl.n_wg * pl.rows * 8);
    pl.off_items = take((size_t) pl.items * 8);
    pl.off_scores = pl.off_lse = 0;
    if (a->weights) {
        pl.off_scores = take((size_t) a->n_seq * a->n_head * a->bt_stride * PAGE * 4);
        pl.off_lse    = take((size_t) a->n_seq * a->n_head * 8);
    }
    pl.bytes = at;
    return pl;
}

// LDS over the 64 KB a kernel gets unasked: granted once a device, whatever it asks for later.
template <typename K> hipError_t launch_lds(K kernel, const AttnP & p, int threads, int lds, std::atomic<uint64_t> & granted, hipStream_t st) {
    if (lds >= 60 * 1024) {                                   // (the kernels' own shared arrays come on top)
        int dev = 0;
        hipError_t e = hipGetDevice(&dev);
        if (e != hipSuccess) return e;
        const uint64_t bit = dev < 64 ? (uint64_t) 1 << dev : 0;
        if (!(granted.load(std::memory_order_relaxed) & bit)) {
            if ((e = hipFuncSetAttribute((const void *) kernel, hipFuncAttributeMaxDynamicSharedMemorySize, lds)) != hipSuccess) return e;
            granted.fetch_or(bit, std::memory_order_relaxed);
        }
    }
    hipLaunchKernelGGL(kernel, dim3((unsigned) p.n_wg), dim3((unsigned) threads), lds, st, p);
    return hipGetLastError();
}
template <bool F16, int DK, int DV, int NB, bool BIAS>
hipError_t launch_main(const AttnP & p, hipStream_t st) {
    static std::atomic<uint64_t> granted{ 0 };
    if constexpr (NB == 1 && DK < 256) if (p.quad) return launch_lds(gqa_attn_kernel<F16, DK, DV, NB, BIAS, true>, p, 256, 0, granted, st);
    return launch_lds(gqa_attn_kernel<F16, DK, DV, NB, BIAS, false>, p, 256, 4 * 16 * DV * 4, granted, st);
}
template <bool F16, bool BIAS>
hipError_t launch_scores(const AttnP & p, hipStream_t st) {
    static_assert(LROWS * LPITCH + LWAVES * LROWS * 8 <= 160 * 1024, "LDS");
    static std::atomic<uint64_t> granted{ 0 };
    return launch_lds(gqa_scores_kernel<F16, BIAS>, p, 64 * LWAVES, LROWS * LPITCH, granted, st);
}

template <bool F16, int NB, bool BIAS>
hipError_t launch_widths(const AttnP & p, int dk, hipStream_t st) {
    switch (dk) {
        case 64:  return launch_main<F16, 64, 64, NB, BIAS>(p, st);
        case 128: return launch_main<F16, 128, 128, NB, BIAS>(p, st);
        case 192: return launch_main<F16, 192, 128, NB, BIAS>(p, st);
        default:
            if constexpr (NB == 1) return launch_main<F16, 256, 256, NB, BIAS>(p, st);
            else                   return hipErrorInvalidValue;        // (make_plan: one block)
    }
}

template <bool F16>
hipError_t launch_all(const AttnP & p, const Plan & pl, int dk, hipStream_t st) {
    const bool bias = p.mask || p.cap_out != 0.f;
    hipError_t e;
    if (dk == LK)        e = bias ? launch_scores<F16, true>(p, st) : launch_scores<F16, false>(p, st);
    else if (pl.nb == 2) e = bias ? launch_widths<F16, 2, true>(p, dk, st) : launch_widths<F16, 2, false>(p, dk, st);
    else                 e = bias ? launch_widths<F16, 1, true>(p, dk, st) : launch_widths<F16, 1, false>(p, dk, st);
    if (e != hipSuccess) return e;
    int joins = p.dv ? p.group : 0;
    const int  groups = p.n_seq * p.n_head_kv;
    const bool ahead  = p.scores && (int64_t) pl.pieces * p.group >= JOIN_AHEAD;
    if (!p.scores || (ahead && joins)) {
        hipLaunchKernelGGL((gqa_join_kernel<F16, 0>), dim3((unsigned) joins, (unsigned) groups), dim3(JOIN), 0, st, p, joins, 0, 0);
        joins = 0;
    } else if (ahead) hipLaunchKernelGGL(gqa_lse_kernel, dim3((unsigned) ((p.group + 3) / 4), (unsigned) groups), dim3(JOIN), 0, st, p);
    if ((e = hipGetLastError()) != hipSuccess || !p.scores) return e;
    int parts = 1;
    while (parts < 16 && parts < p.group) parts *= 2;
    const int64_t blocks = (p.cap * parts + 4 * JOIN - 1) / (4 * JOIN), share = (SUM_BLOCKS + groups - 1) / groups;
    const dim3 grid((unsigned) (joins + (blocks < share ? blocks : share)), (unsigned) groups);
    if (p.group <= parts) hipLaunchKernelGGL((gqa_join_kernel<F16, 1>), grid, dim3(JOIN), 0, st, p, joins, parts, (int) ahead);
    else                  hipLaunchKernelGGL((gqa_join_kernel<F16, 8>), grid, dim3(JOIN), 0, st, p, joins, parts, (int) ahead);
    return hipGetLastError();
}

int check_pool(const gqa_pool & c) {
    if (!c.data) return MLA_ERR_NULL;
    if (!al16(c.data) || (c.nb_page & 15) || (c.nb_row & 15) || (c.nb_head & 15)) return MLA_ERR_BAD_ALIGNMENT;
    if (c.nb_page < 0 || c.nb_head < 0 || c.nb_row < 0 || c.nb_row > (1 << 23) || c.nb_page >= ((int64_t) 1 << 32)) return MLA_ERR_BAD_SHAPE;   // 128 rows within 31 bits, a page within 32
    return 0;
}

}  // namespace

extern "C" int gqa_attn_check(const gqa_attn_args * a) {
    if (!a) return MLA_ERR_NULL;
    if (a->kv_type != MLA_TYPE_BF16 && a->kv_type != MLA_TYPE_F16) return MLA_ERR_BAD_TYPE;
    if ((a->q_type != MLA_TYPE_F32 && a->q_type != a->kv_type) || (a->dst_type != MLA_TYPE_F32 && a->dst_type != a->kv_type)) return MLA_ERR_BAD_TYPE;
    if (a->n_seq < 0 || a->n_head < 1 || a->n_head_kv < 1 || a->n_head % a->n_head_kv || a->window < 0 || a->n_workgroups < 0 || a->n_workgroups > 65536) return MLA_ERR_BAD_SHAPE;
    const bool widths = a->dk == 64 || a->dk == 128 || a->dk == 256 ? a->dv == a->dk : (a->dk == 192 && a->dv == 128) || (a->dk == LK && a->dv == 0 && a->n_head_kv == 1);
    if (!widths) return MLA_ERR_UNSUPPORTED;
    if (!(a->logit_softcap >= 0.f && a->logit_softcap <= FLT_MAX)) return MLA_ERR_UNSUPPORTED;
    if (a->n_seq == 0) return 0;
    if (!a->q || !a->block_table || !a->seq_lens) return MLA_ERR_NULL;
    if (a->n_pages < 1 || a->bt_stride < 1) return MLA_ERR_BAD_SHAPE;
    // rows are counted in 30 bits, units of work and workgroups in 31
    const int64_t lim = (int64_t) 1 << 31;
    if (a->bt_stride >= lim / 2 / PAGE || (int64_t) a->n_seq * a->n_head >= (1 << 24) || (int64_t) a->n_seq * a->n_head_kv > 65535 || (int64_t) a->n_seq * a->n_head * a->bt_stride >= lim)
        return MLA_ERR_BAD_SHAPE;
    if (a->n_head / a->n_head_kv + SUM_BLOCKS >= (1 << 24)) return MLA_ERR_BAD_SHAPE;        // (the last launch: fewer than 2^32 threads, and nothing starts of a call whose last could not)
    int rc = check_pool(a->k);
    if (rc) return rc;
    if (a->dv) {
        if ((rc = check_pool(a->v))) return rc;
        if (!a->dst) return MLA_ERR_NULL;
        const int al = a->dst_type == MLA_TYPE_F32 ? 15 : 7;
        if (((uintptr_t) a->dst & al) || (a->d_nb1 & al) || (a->d_nb2 & al)) return MLA_ERR_BAD_ALIGNMENT;
    } else if (a->v.data || a->dst) return MLA_ERR_UNSUPPORTED;
    else if (!a->weights) return MLA_ERR_NULL;
    if (!al16(a->q) || (a->q_nb1 & 15) || (a->q_nb2 & 15)) return MLA_ERR_BAD_ALIGNMENT;
    if (a->mask) {
        if (((uintptr_t) a->mask & 1) || (a->mask_nb1 & 1)) return MLA_ERR_BAD_ALIGNMENT;
        if (a->mask_ne0 < 0) return MLA_ERR_BAD_SHAPE;
    }
    // what is written is nothing that is read (by its address alone: strides may lay one between the other's rows)
    for (const void * w : { (const void *) a->dst, (const void *) a->weights })
        if (w && (w == a->q || w == a->k.data || w == a->v.data || w == a->mask || w == (const void *) a->seq_lens || w == (const void *) a->block_table)) return MLA_ERR_UNSUPPORTED;
    if (a->dst && a->dst == a->weights) return MLA_ERR_UNSUPPORTED;
    if (a->weights && (((uintptr_t) a->weights & 3) || (a->w_nb1 & 3) || (a->w_nb2 & 3))) return MLA_ERR_BAD_ALIGNMENT;
    return 0;
}

extern "C" size_t gqa_attn_workspace_size(const gqa_attn_args * a) {
    if (gqa_attn_check(a) || a->n_seq == 0) return 0;
    return make_plan(a).bytes;
}

extern "C" int gqa_attn_launch(const gqa_attn_args * a, void * stream) {
    const int rc = gqa_attn_check(a);
    if (rc) return rc;
    if (a->n_seq == 0) return 0;
    const Plan pl = make_plan(a);
    if (!a->workspace || ((uintptr_t) a->workspace & 255) || a->workspace_size < pl.bytes) return MLA_ERR_WORKSPACE;
    char * ws = (char *) a->workspace;
    AttnP  p;
    p.q = (const char *) a->q; p.q_nb1 = a->q_nb1; p.q_nb2 = a->q_nb2; p.q_f32 = a->q_type == MLA_TYPE_F32;
    p.k = (const char *) a->k.data; p.k_page = (unsigned) a->k.nb_page; p.k_head = a->k.nb_head; p.k_row = (int) a->k.nb_row;
    p.v = (const char *) a->v.data; p.v_page = (unsigned) a->v.nb_page; p.v_head = a->v.nb_head; p.v_row = (int) a->v.nb_row;
    p.n_pages = a->n_pages; p.block_table = a->block_table; p.bt_stride = a->bt_stride; p.seq_lens = a->seq_lens;
    p.mask = (const char *) a->mask; p.mask_nb1 = a->mask_nb1;
    p.mask_len = a->mask && a->mask_ne0 < a->bt_stride * PAGE ? (int) a->mask_ne0 : (int) (a->bt_stride * PAGE);
    p.weights = a->weights; p.w_nb1 = a->w_nb1; p.w_nb2 = a->w_nb2;
    p.dst = (char *) a->dst; p.d_nb1 = a->d_nb1; p.d_nb2 = a->d_nb2; p.dst_f32 = a->dst_type == MLA_TYPE_F32;
    p.scale_log2 = a->scale * LOG2E;
    // (a cap so small or large that these leave f32: the largest number does the same)
    p.cap_in  = a->logit_softcap > 0.f ? fminf(fmaxf(a->scale / a->logit_softcap, -FLT_MAX), FLT_MAX) : 0.f;
    p.cap_out = fminf(a->logit_softcap * LOG2E, FLT_MAX);
    p.window = a->window; p.n_seq = a->n_seq; p.n_head = a->n_head; p.n_head_kv = a->n_head_kv; p.group = a->n_head / a->n_head_kv;
    p.row_blocks = pl.row_blocks; p.head_blocks = pl.head_blocks; p.rows = pl.rows; p.quad = pl.quad; p.dv = a->dv; p.n_wg = pl.n_wg;
    p.part_o = (float *) ws; p.part_ml = (float2 *) (ws + pl.off_ml); p.items = (int2 *) (ws + pl.off_items);
    p.scores = a->weights ? (float *) (ws + pl.off_scores) : nullptr; p.lse = a->weights ? (float2 *) (ws + pl.off_lse) : nullptr;
    p.cap = a->bt_stride * PAGE;
    return (int) (a->kv_type == MLA_TYPE_F16 ? launch_all<true>(p, pl, a->dk, (hipStream_t) stream) : launch_all<false>(p, pl, a->dk, (hipStream_t) stream));
}
