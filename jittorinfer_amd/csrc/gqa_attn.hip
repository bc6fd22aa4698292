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
//   * P goes in as two 16-bit numbers, hi + lo: the matrix cores are idle otherwise, and P rounded once (2^-9 in bf16) would be the
//     largest error of the whole pass.
//   * the running maximum moves only when a score passes it by more than 2^8 (exp2 sums then reach 2^8 a key, far from f32's range), so
//     the common tile has no reduction across lanes and no rescaling.
//   * K of the next tile is requested when this tile's scores are done, V when its products are.
//
// Work: the list of all (sequence, KV head, page) units, in that order, is dealt to the workgroups in equal runs, from the lengths on
// the device (nothing on the host depends on them, so a captured launch stays valid while they change).  A run that covers a (sequence,
// KV head) whole writes its result; the others leave (o, m, l) in f32 for the second kernel, which joins them in the order of the rows.
// With weights the first kernel also leaves every score, 4 bytes a (head, row), and a third one adds exp(s - m) / l over the group.

#include <math.h>

#include "mla_common.hpp"
#include "../../include/gqa_attn.h"

using namespace mla;

namespace {

struct AttnP {
    const char * q; int64_t q_nb1, q_nb2; int q_f32;
    const char * k; int64_t k_page, k_head; int k_row;
    const char * v; int64_t v_page, v_head; int v_row;
    int64_t n_pages;
    const int32_t * block_table; int64_t bt_stride;
    const int32_t * seq_lens;
    const char * mask; int64_t mask_nb1, mask_ne0;
    float * weights; int64_t w_nb1, w_nb2;
    char * dst; int64_t d_nb1, d_nb2; int dst_f32;
    float scale_log2;             // scale * log2(e)
    float cap_in, cap_out;        // soft cap c: c * tanh(x / c) = c - 2c / (exp2(cap_in * q.k) + 1), times log2(e); cap_out = 0: none
    int window, n_seq, n_head, n_head_kv, group, row_blocks, head_blocks, dv;
    int n_wg;
    float *  part_o;              // [2 * n_wg][rows][DV]
    float2 * part_ml;             // [2 * n_wg][rows]: maximum (log2 units), sum
    int2 *   items;               // [n_seq * head_blocks]: (2 * first workgroup + whether the item begins inside its run, last workgroup)
    float *  scores;              // [n_seq][n_head][cap] in log2 units, or nullptr
    float2 * lse;                 // [n_seq][n_head]: maximum, 1 / sum
    int64_t  cap;                 // bt_stride * 128
};

constexpr int PAGE = MLA_PAGE_TOKENS;

// Workgroups a CU holds: a wave's tile of K and V, its Q fragments and its accumulators take up to 256 registers for heads up to 128 wide
// and one block of 16 query heads, more (two waves a SIMD would spill) beyond.
constexpr int wg_per_cu(int dk, int nb) { return dk <= 64 || (dk <= 192 && nb == 1) ? 2 : 1; }

template <bool F16> __device__ __forceinline__ f32x4 mfma16(u32x4 a, u32x4 b, f32x4 c) {
    if constexpr (F16) return __builtin_amdgcn_mfma_f32_16x16x32_f16(bitcast<f16x8>(a), bitcast<f16x8>(b), c, 0, 0, 0);
    else               return __builtin_amdgcn_mfma_f32_16x16x32_bf16(bitcast<bf16x8>(a), bitcast<bf16x8>(b), c, 0, 0, 0);
}
template <bool F16> __device__ __forceinline__ unsigned short to16(float f) {
    if constexpr (F16) return bitcast<unsigned short>((_Float16) f);
    else               return bitcast<unsigned short>((__bf16) f);
}
template <bool F16> __device__ __forceinline__ float from16(unsigned short h) {
    if constexpr (F16) return (float) bitcast<_Float16>(h);
    else               return __uint_as_float((unsigned) h << 16);
}

// The rows a sequence attends to, [first, last).
struct Span { int first, last; };
__device__ __forceinline__ Span span_of(const AttnP & p, int b) {
    int64_t n = p.seq_lens[b];
    n = n < 0 ? 0 : n > p.cap ? p.cap : n;
    const int64_t first = p.window > 0 && n > p.window ? n - p.window : 0;
    if (p.mask && n > p.mask_ne0) n = p.mask_ne0;
    return n > first ? Span{ (int) first, (int) n } : Span{ 0, 0 };
}
__device__ __forceinline__ int pages_of(Span s) { return s.last > s.first ? (s.last + PAGE - 1) / PAGE - s.first / PAGE : 0; }

__device__ __forceinline__ int wave_sum(int v) {
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) v += __shfl_xor(v, d, 64);
    return v;
}

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

// threads 256 = 4 waves; wave w takes quarter w of every page of the run.
template <bool F16, int DK, int DV, int NB, bool BIAS>
__global__ void __launch_bounds__(256, wg_per_cu(DK, NB)) gqa_attn_kernel(const AttnP p) {
    constexpr int  KC    = DK / 32;
    constexpr bool Q_LDS = DK > 256;                    // 18 operand fragments a head block: shared by the waves out of LDS
    constexpr int  QP    = DK * 2 + 16;                 // its row pitch
    constexpr int  ROWS  = NB * 16;
    using VG = VGeom<DV ? DV : 64>;
    extern __shared__ __attribute__((aligned(16))) char lds[];
    __shared__ int    sh_total, sh_seq, sh_before, sh_part[4];
    __shared__ float2 sh_ml[4][ROWS];

    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, l15 = lane & 15, lg = lane >> 4;
    const int wg = blockIdx.x;

    // ---- which units are this workgroup's
    if (threadIdx.x == 0) sh_total = 0;
    __syncthreads();
    {
        int mine = 0;
        for (int b = threadIdx.x; b < p.n_seq; b += 256) mine += pages_of(span_of(p, b));
        mine = wave_sum(mine);
        if (lane == 0 && mine) atomicAdd(&sh_total, mine);   // (integers: any order)
    }
    __syncthreads();
    const int  total = sh_total * p.head_blocks;
    const Deal deal{ total / p.n_wg, total % p.n_wg };
    int        u = run_start(deal, wg);
    const int  u_end = run_start(deal, wg + 1);
    if (u >= u_end) return;
    {
        int before = 0;
        for (int b0 = 0; b0 < p.n_seq; b0 += 256) {
            const int b = b0 + (int) threadIdx.x;
            const int n = b < p.n_seq ? pages_of(span_of(p, b)) * p.head_blocks : 0;
            int incl = n;
#pragma unroll
            for (int d = 1; d < 64; d <<= 1) { const int o = __shfl_up(incl, d, 64); if (lane >= d) incl += o; }
            if (lane == 63) sh_part[wave] = incl;
            __syncthreads();
            int ahead = before;
            for (int w = 0; w < wave; w++) ahead += sh_part[w];
            if (n > 0 && u >= ahead + incl - n && u < ahead + incl) { sh_seq = b; sh_before = ahead + incl - n; }
            before += sh_part[0] + sh_part[1] + sh_part[2] + sh_part[3];
            __syncthreads();
            if (u < before) break;
        }
    }
    int  b = sh_seq;
    Span s = span_of(p, b);
    int  np = pages_of(s);
    int  hb = (u - sh_before) / np, pg = (u - sh_before) % np;

    for (bool fresh = true; u < u_end; fresh = false) {
        const int  n = min(np - pg, u_end - u);              // pages of this piece
        const bool begins = pg == 0, whole = begins && n == np;
        const int  kvh = hb / p.row_blocks, row0 = (hb - kvh * p.row_blocks) * ROWS;   // first head of the group taken here
        const int  heads = min(ROWS, p.group - row0);
        const int  head0 = kvh * p.group + row0;
        if (begins && threadIdx.x == 0) p.items[(int64_t) b * p.head_blocks + hb] = make_int2(2 * wg + (fresh ? 0 : 1), owner_of(deal, u + np - 1));

        // ---- Q: operand fragments, lane (h, g) k = 32 c + 8 g .. + 7; heads past the group: zeros
        u32x4 qf[Q_LDS ? 1 : NB * KC];
        auto q_frag = [&](int row, int off) -> u32x4 {       // 8 values from value `off` on
            if (row >= heads) return u32x4{ 0u, 0u, 0u, 0u };
            const char * src = p.q + (int64_t) b * p.q_nb2 + (int64_t) (head0 + row) * p.q_nb1;
            if (!p.q_f32) return *(const u32x4 *) (src + off * 2);
            const f32x4 x = *(const f32x4 *) (src + off * 4), y = *(const f32x4 *) (src + off * 4 + 16);
            return u32x4{ pack2<F16>(x.x, x.y), pack2<F16>(x.z, x.w), pack2<F16>(y.x, y.y), pack2<F16>(y.z, y.w) };
        };
        if constexpr (Q_LDS) {
            for (int i = threadIdx.x; i < ROWS * (DK / 8); i += 256) {
                const int row = i / (DK / 8), c = i - row * (DK / 8);
                *(u32x4 *) (lds + row * QP + c * 16) = q_frag(row, c * 8);
            }
            __syncthreads();
        } else {
#pragma unroll
            for (int nb = 0; nb < NB; nb++)
#pragma unroll
                for (int c = 0; c < KC; c++) qf[nb * KC + c] = q_frag(nb * 16 + l15, c * 32 + lg * 8);
        }

        float m[NB], l[NB];
        f32x4 acc[NB][DV ? VG::COLS : 1];
#pragma unroll
        for (int nb = 0; nb < NB; nb++) {
            m[nb] = -INFINITY; l[nb] = 0.f;
#pragma unroll
            for (int c = 0; c < (DV ? VG::COLS : 1); c++) acc[nb][c] = f32x4{ 0.f, 0.f, 0.f, 0.f };
        }

        const int32_t * bt = p.block_table + (int64_t) b * p.bt_stride + s.first / PAGE + pg;
        const int       t_page0 = (s.first / PAGE + pg) * PAGE;
        u32x4 kf[2][KC];
        u32x2 vf[8][DV ? VG::COLS / 4 : 1];
        // the slots in the page whose rows a lane loads: rows outside the span are replaced by the nearest one inside
        auto slot = [&](int i, int r) { return min(max(wave * 32 + r, s.first - (t_page0 + i * PAGE)), s.last - 1 - (t_page0 + i * PAGE)); };
        auto load_k = [&](int i, int64_t page) {
            const char * base = p.k + page * p.k_page + (int64_t) kvh * p.k_head;
#pragma unroll
            for (int blk = 0; blk < 2; blk++) {
                const char * row = base + slot(i, blk * 16 + l15) * p.k_row + lg * 16;
#pragma unroll
                for (int c = 0; c < KC; c++) kf[blk][c] = *(const u32x4 *) (row + c * 64);
            }
        };
        auto load_v = [&](int i, int64_t page) {
            if constexpr (DV > 0) {
                const char * base = p.v + page * p.v_page + (int64_t) kvh * p.v_head;
#pragma unroll
                for (int e = 0; e < 8; e++) {
                    const char * row = base + slot(i, (e >> 2) * 16 + lg * 4 + (e & 3)) * p.v_row + l15 * (VG::W * 2);
#pragma unroll
                    for (int gr = 0; gr < VG::GROUPS; gr++) {
                        if constexpr (VG::W == 8) {
                            const u32x4 x = *(const u32x4 *) (row + gr * 256);
                            vf[e][2 * gr] = u32x2{ x[0], x[1] }; vf[e][2 * gr + 1] = u32x2{ x[2], x[3] };
                        } else vf[e][gr] = *(const u32x2 *) row;
                    }
                }
            }
        };
        auto page_at = [&](int i, bool & ok) -> int64_t {      // page of the piece's page i; a bad id: page 0 is read, not used
            const int id = bt[i];
            ok = id >= 0 && id < p.n_pages;
            return ok ? id : 0;
        };

        bool    ok;
        int64_t page = page_at(0, ok);
        load_k(0, page);
        load_v(0, page);
        for (int i = 0; i < n; i++) {
            const int  t0 = t_page0 + i * PAGE + wave * 32;     // first row of the tile
            const int  lo = max(s.first - t0, 0), hi = min(s.last - t0, 32);
            const bool use = ok && hi > lo, all = lo == 0 && hi == 32;
            bool       ok_next = false;
            const int64_t next = i + 1 < n ? page_at(i + 1, ok_next) : 0;

            f32x4 sc[NB][2];
#pragma unroll
            for (int nb = 0; nb < NB; nb++) {
                sc[nb][0] = f32x4{ 0.f, 0.f, 0.f, 0.f }; sc[nb][1] = sc[nb][0];
#pragma unroll
                for (int c = 0; c < KC; c++) {
                    u32x4 qq;
                    if constexpr (Q_LDS) qq = *(const u32x4 *) (lds + (nb * 16 + l15) * QP + c * 64 + lg * 16);
                    else                 qq = qf[nb * KC + c];
                    sc[nb][0] = mfma16<F16>(kf[0][c], qq, sc[nb][0]);
                    sc[nb][1] = mfma16<F16>(kf[1][c], qq, sc[nb][1]);
                }
            }
            if (i + 1 < n) load_k(i + 1, next);

            // scores in log2 units
            float mk[2][4];
            bool  out[2][4];
            if constexpr (BIAS) {
#pragma unroll
                for (int blk = 0; blk < 2; blk++)
#pragma unroll
                    for (int j = 0; j < 4; j++) {
                        const int r = blk * 16 + lg * 4 + j;
                        mk[blk][j] = 0.f; out[blk][j] = true;          // (rows outside the span repeat one inside, which may be masked)
                        if (p.mask && r >= lo && r < hi) {
                            const float x = f16_bits_to_f32(*(const unsigned short *) (p.mask + (int64_t) b * p.mask_nb1 + (int64_t) (t0 + r) * 2));
                            out[blk][j] = x == -INFINITY;
                            mk[blk][j]  = x * LOG2E;
                        }
                    }
            }
            float x[NB][2][4];
#pragma unroll
            for (int nb = 0; nb < NB; nb++)
#pragma unroll
                for (int blk = 0; blk < 2; blk++)
#pragma unroll
                    for (int j = 0; j < 4; j++) {
                        float y;
                        if constexpr (BIAS) {
                            if (p.cap_out != 0.f) y = p.cap_out - 2.f * p.cap_out * __builtin_amdgcn_rcpf(fast_exp2(p.cap_in * sc[nb][blk][j]) + 1.f);
                            else                  y = p.scale_log2 * sc[nb][blk][j];
                            if (p.mask) y = out[blk][j] ? -INFINITY : y + mk[blk][j];
                        } else y = p.scale_log2 * sc[nb][blk][j];
                        x[nb][blk][j] = y;
                    }
            if (!use || !all) {
#pragma unroll
                for (int nb = 0; nb < NB; nb++)
#pragma unroll
                    for (int blk = 0; blk < 2; blk++)
#pragma unroll
                        for (int j = 0; j < 4; j++) {
                            const int r = blk * 16 + lg * 4 + j;
                            if (!use || r < lo || r >= hi) x[nb][blk][j] = -INFINITY;
                        }
            }
            if (p.scores) {
#pragma unroll
                for (int nb = 0; nb < NB; nb++)
                    if (nb * 16 + l15 < heads) {
                        float * to = p.scores + ((int64_t) b * p.n_head + head0 + nb * 16 + l15) * p.cap + t0 + lg * 4;
                        *(f32x4 *) to        = f32x4{ x[nb][0][0], x[nb][0][1], x[nb][0][2], x[nb][0][3] };
                        *(f32x4 *) (to + 16) = f32x4{ x[nb][1][0], x[nb][1][1], x[nb][1][2], x[nb][1][3] };
                    }
            }
            if (use) {
                u32x4 ph[NB], pl[NB];
#pragma unroll
                for (int nb = 0; nb < NB; nb++) {
                    float top = x[nb][0][0];
#pragma unroll
                    for (int e = 1; e < 8; e++) top = fmaxf(top, x[nb][e >> 2][e & 3]);
                    if (__any(top > m[nb] + 8.f)) {
                        top = fmaxf(top, __shfl_xor(top, 16, 64));
                        top = fmaxf(top, __shfl_xor(top, 32, 64));
                        const float nm = fmaxf(top, m[nb]);
                        const float a  = m[nb] == nm ? 1.f : fast_exp2(m[nb] - nm);
                        m[nb] = nm;
                        l[nb] *= a;
                        if constexpr (DV > 0) {
#pragma unroll
                            for (int j = 0; j < 4; j++) {
                                const float aj = __shfl(a, lg * 4 + j, 64);
#pragma unroll
                                for (int c = 0; c < VG::COLS; c++) acc[nb][c][j] *= aj;
                            }
                        }
                    }
                    const float mm = m[nb] == -INFINITY ? 0.f : m[nb];
                    float e8[8];
#pragma unroll
                    for (int e = 0; e < 8; e++) { e8[e] = fast_exp2(x[nb][e >> 2][e & 3] - mm); l[nb] += e8[e]; }
                    if constexpr (DV > 0) {
#pragma unroll
                        for (int e = 0; e < 4; e++) {
                            const unsigned short h0 = to16<F16>(e8[2 * e]), h1 = to16<F16>(e8[2 * e + 1]);
                            ph[nb][e] = h0 | ((unsigned) h1 << 16);
                            pl[nb][e] = to16<F16>(e8[2 * e] - from16<F16>(h0)) | ((unsigned) to16<F16>(e8[2 * e + 1] - from16<F16>(h1)) << 16);
                        }
                    }
                }
                if constexpr (DV > 0) {
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
                        for (int nb = 0; nb < NB; nb++) {
                            acc[nb][c] = mfma16<F16>(ph[nb], bf, acc[nb][c]);
                            acc[nb][c] = mfma16<F16>(pl[nb], bf, acc[nb][c]);
                        }
                    }
                }
            }
            if (i + 1 < n) load_v(i + 1, next);
            page = next; ok = ok_next;
        }

        // ---- the four waves' results meet in LDS
#pragma unroll
        for (int nb = 0; nb < NB; nb++) {
            float t = l[nb];
            t += __shfl_xor(t, 16, 64);
            t += __shfl_xor(t, 32, 64);
            if (lg == 0) sh_ml[wave][nb * 16 + l15] = make_float2(m[nb], t);
        }
        __syncthreads();
        auto joined = [&](int row) -> float2 {               // maximum and sum over the waves
            float M = -INFINITY, L = 0.f;
#pragma unroll
            for (int w = 0; w < 4; w++) M = fmaxf(M, sh_ml[w][row].x);
#pragma unroll
            for (int w = 0; w < 4; w++) L += sh_ml[w][row].y == 0.f ? 0.f : sh_ml[w][row].y * fast_exp2(sh_ml[w][row].x - M);
            return make_float2(M, L);
        };
        const int64_t piece = 2 * (int64_t) wg + (fresh ? 0 : 1);
        for (int r = threadIdx.x; r < heads; r += 256) {
            const float2 ml = joined(r);
            if (!whole) p.part_ml[piece * ROWS + r] = ml;
            else if (p.scores) p.lse[(int64_t) b * p.n_head + head0 + r] = make_float2(ml.x == -INFINITY ? 0.f : ml.x, ml.y == 0.f ? 0.f : 1.f / ml.y);
        }
        if constexpr (DV > 0) {
            float * tile = (float *) lds;                     // [4][16][DV]
#pragma unroll
            for (int nb = 0; nb < NB; nb++) {
                if (nb) __syncthreads();
#pragma unroll
                for (int j = 0; j < 4; j++) {
                    const int    row = nb * 16 + lg * 4 + j;
                    const float  mw  = sh_ml[wave][row].x;
                    const float2 ml  = joined(row);
                    const float  f   = mw == -INFINITY ? 0.f : fast_exp2(mw - ml.x);
                    float * to = tile + (wave * 16 + lg * 4 + j) * DV + l15 * VG::W;
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
                    f32x4 o = *(const f32x4 *) (tile + r * DV + c);
#pragma unroll
                    for (int w = 1; w < 4; w++) o += *(const f32x4 *) (tile + (w * 16 + r) * DV + c);
                    if (!whole) *(f32x4 *) (p.part_o + (piece * ROWS + row) * DV + c) = o;
                    else {
                        const float L = joined(row).y, inv = L == 0.f ? 0.f : 1.f / L;   // (a NaN stays one)
                        char * to = p.dst + (int64_t) b * p.d_nb2 + (int64_t) (head0 + row) * p.d_nb1;
                        o *= inv;
                        if (p.dst_f32) *(f32x4 *) (to + c * 4) = o;
                        else *(u32x2 *) (to + c * 2) = u32x2{ to16<F16>(o.x) | ((unsigned) to16<F16>(o.y) << 16), to16<F16>(o.z) | ((unsigned) to16<F16>(o.w) << 16) };
                    }
                }
            }
        }
        __syncthreads();                                      // LDS is free again for the next piece

        u += n; pg = 0;
        if (++hb == p.head_blocks && u < u_end) {
            hb = 0;
            do { b++; s = span_of(p, b); np = pages_of(s); } while (np == 0);   // (u < u_end <= total: there is such a sequence)
        }
    }
}

// Joins what the runs left of one head (grid: a workgroup per (sequence, head)): o = sum_i o_i 2^(m_i - M) / sum_i l_i 2^(m_i - M), pieces in
// the order of the rows.  Heads whose rows one run covered are done; heads without a row get zeros.
template <bool F16>
__global__ void __launch_bounds__(256) gqa_join_kernel(const AttnP p, const int rows) {
    __shared__ float  red[8];
    __shared__ f32x4  sum[256];
    const int b = blockIdx.x / p.n_head, h = blockIdx.x - b * p.n_head;
    const int kvh = h / p.group, r_all = h - kvh * p.group, rb = r_all / rows, row = r_all - rb * rows;
    char *    dst = p.dst ? p.dst + (int64_t) b * p.d_nb2 + (int64_t) h * p.d_nb1 : nullptr;
    const int cols = p.dv / 4;                                // runs of 4 columns
    auto store = [&](int c, f32x4 o) {
        if (p.dst_f32) *(f32x4 *) (dst + c * 16) = o;
        else *(u32x2 *) (dst + c * 8) = u32x2{ to16<F16>(o.x) | ((unsigned) to16<F16>(o.y) << 16), to16<F16>(o.z) | ((unsigned) to16<F16>(o.w) << 16) };
    };
    if (pages_of(span_of(p, b)) == 0) {
        for (int c = threadIdx.x; c < cols; c += 256) store(c, f32x4{ 0.f, 0.f, 0.f, 0.f });
        return;
    }
    const int2 it = p.items[(int64_t) b * p.head_blocks + kvh * p.row_blocks + rb];
    const int  v0 = it.x >> 1, n = it.y - v0 + 1;
    if (n == 1) return;
    auto slot = [&](int i) -> int64_t { return ((int64_t) (i ? 2 * (v0 + i) : it.x)) * rows + row; };

    float M = -INFINITY;
    for (int i = threadIdx.x; i < n; i += 256) M = fmaxf(M, p.part_ml[slot(i)].x);
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) M = fmaxf(M, __shfl_xor(M, d, 64));
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = M;
    __syncthreads();
    M = fmaxf(fmaxf(red[0], red[1]), fmaxf(red[2], red[3]));
    float L = 0.f;
    for (int i = threadIdx.x; i < n; i += 256) { const float2 ml = p.part_ml[slot(i)]; if (ml.y != 0.f) L += ml.y * fast_exp2(ml.x - M); }
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) L += __shfl_xor(L, d, 64);
    if ((threadIdx.x & 63) == 0) red[4 + (threadIdx.x >> 6)] = L;
    __syncthreads();
    L = (red[4] + red[5]) + (red[6] + red[7]);
    const float inv = L == 0.f ? 0.f : 1.f / L;
    if (p.scores && threadIdx.x == 0) p.lse[(int64_t) b * p.n_head + h] = make_float2(M == -INFINITY ? 0.f : M, inv);
    if (!cols) return;

    const int groups = 256 / cols, g = threadIdx.x / cols, c = threadIdx.x - g * cols;   // (cols: 16, 32 or 64)
    f32x4 o = { 0.f, 0.f, 0.f, 0.f };
    for (int i = g; i < n; i += groups) {
        const int64_t at = slot(i);
        const float2  ml = p.part_ml[at];
        if (ml.y != 0.f) o += *(const f32x4 *) (p.part_o + at * p.dv + c * 4) * fast_exp2(ml.x - M);
    }
    sum[threadIdx.x] = o;
    __syncthreads();
    if (g == 0) {
        for (int i = 1; i < groups; i++) o += sum[i * cols + c];
        store(c, o * inv);
    }
}

// weights[b][g][i] += sum over the group's heads of exp2(s - m) / l, from the scores the first kernel left: 4 rows a thread.
__global__ void __launch_bounds__(256) gqa_weights_kernel(const AttnP p) {
    const int  b = blockIdx.y / p.n_head_kv, kvh = blockIdx.y - b * p.n_head_kv;
    const Span s = span_of(p, b);
    const int  t = (int) (blockIdx.x * 1024 + threadIdx.x * 4);
    if (t >= s.last || t + 4 <= s.first) return;
    const int64_t h0 = (int64_t) b * p.n_head + (int64_t) kvh * p.group;
    f32x4 w = { 0.f, 0.f, 0.f, 0.f };
    for (int h = 0; h < p.group; h++) {
        const float2 ml = p.lse[h0 + h];
        const f32x4  x  = *(const f32x4 *) (p.scores + (h0 + h) * p.cap + t);
#pragma unroll
        for (int j = 0; j < 4; j++) w[j] += fast_exp2(x[j] - ml.x) * ml.y;
    }
    float * to = (float *) ((char *) p.weights + (int64_t) b * p.w_nb2 + (int64_t) kvh * p.w_nb1) + t;
#pragma unroll
    for (int j = 0; j < 4; j++) if (t + j >= s.first && t + j < s.last) to[j] += w[j];
}

// ---------------------------------------------------------------- host

bool al16(const void * ptr) { return ((uintptr_t) ptr & 15) == 0; }

struct Plan {
    int     nb, rows, row_blocks, n_wg;
    int64_t items;
    size_t  off_ml, off_items, off_scores, off_lse, bytes;    // of the workspace; partial rows first
};

Plan make_plan(const gqa_attn_args * a) {
    Plan pl;
    const int group = a->n_head / a->n_head_kv;
    pl.nb = a->dv == 0 ? 8 : group > 16 ? 2 : 1;              // 16 heads a block of the operand; two where the group fills them
    pl.rows = pl.nb * 16;
    pl.row_blocks = (group + pl.rows - 1) / pl.rows;
    pl.items = (int64_t) a->n_seq * a->n_head_kv * pl.row_blocks;
    const int64_t units = pl.items * a->bt_stride;
    const int fill = 256 * wg_per_cu(a->dk, pl.nb);
    pl.n_wg = (int) (units < fill ? units : fill);
    if (a->n_workgroups > 0) pl.n_wg = (int) (units < a->n_workgroups ? units : a->n_workgroups);
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

template <bool F16, int DK, int DV, int NB, bool BIAS>
hipError_t launch_main(const AttnP & p, hipStream_t st) {
    constexpr int lds = DV ? 4 * 16 * DV * 4 : NB * 16 * (DK * 2 + 16);
    static_assert(lds <= 160 * 1024 - 8192, "LDS");
    if (lds > 64 * 1024) {
        const hipError_t e = hipFuncSetAttribute((const void *) gqa_attn_kernel<F16, DK, DV, NB, BIAS>, hipFuncAttributeMaxDynamicSharedMemorySize, lds);
        if (e != hipSuccess) return e;
    }
    hipLaunchKernelGGL((gqa_attn_kernel<F16, DK, DV, NB, BIAS>), dim3((unsigned) p.n_wg), dim3(256), lds, st, p);
    return hipGetLastError();
}

template <bool F16, int NB, bool BIAS>
hipError_t launch_widths(const AttnP & p, int dk, hipStream_t st) {
    switch (dk) {
        case 64:  return launch_main<F16, 64, 64, NB, BIAS>(p, st);
        case 128: return launch_main<F16, 128, 128, NB, BIAS>(p, st);
        case 192: return launch_main<F16, 192, 128, NB, BIAS>(p, st);
        default:  return launch_main<F16, 256, 256, NB, BIAS>(p, st);
    }
}

template <bool F16>
hipError_t launch_all(const AttnP & p, const Plan & pl, int dk, hipStream_t st) {
    const bool bias = p.mask || p.cap_out != 0.f;
    hipError_t e;
    if (dk == 576)       e = bias ? launch_main<F16, 576, 0, 8, true>(p, st) : launch_main<F16, 576, 0, 8, false>(p, st);
    else if (pl.nb == 2) e = bias ? launch_widths<F16, 2, true>(p, dk, st) : launch_widths<F16, 2, false>(p, dk, st);
    else                 e = bias ? launch_widths<F16, 1, true>(p, dk, st) : launch_widths<F16, 1, false>(p, dk, st);
    if (e != hipSuccess) return e;
    hipLaunchKernelGGL((gqa_join_kernel<F16>), dim3((unsigned) (p.n_seq * p.n_head)), dim3(256), 0, st, p, pl.rows);
    if ((e = hipGetLastError()) != hipSuccess || !p.scores) return e;
    hipLaunchKernelGGL(gqa_weights_kernel, dim3((unsigned) ((p.cap + 1023) / 1024), (unsigned) (p.n_seq * p.n_head_kv)), dim3(256), 0, st, p);
    return hipGetLastError();
}

int check_pool(const gqa_pool & c) {
    if (!c.data) return MLA_ERR_NULL;
    if (!al16(c.data) || (c.nb_page & 15) || (c.nb_row & 15) || (c.nb_head & 15)) return MLA_ERR_BAD_ALIGNMENT;
    if (c.nb_page < 0 || c.nb_head < 0 || c.nb_row < 0 || c.nb_row > (1 << 23)) return MLA_ERR_BAD_SHAPE;   // 128 rows within 31 bits
    return 0;
}

}  // namespace

extern "C" int gqa_attn_check(const gqa_attn_args * a) {
    if (!a) return MLA_ERR_NULL;
    if (a->kv_type != MLA_TYPE_BF16 && a->kv_type != MLA_TYPE_F16) return MLA_ERR_BAD_TYPE;
    if ((a->q_type != MLA_TYPE_F32 && a->q_type != a->kv_type) || (a->dst_type != MLA_TYPE_F32 && a->dst_type != a->kv_type)) return MLA_ERR_BAD_TYPE;
    if (a->n_seq < 0 || a->n_head < 1 || a->n_head_kv < 1 || a->n_head % a->n_head_kv || a->window < 0 || a->n_workgroups < 0 || a->n_workgroups > 65536) return MLA_ERR_BAD_SHAPE;
    const bool widths = a->dk == 64 || a->dk == 128 || a->dk == 256 ? a->dv == a->dk : (a->dk == 192 && a->dv == 128) || (a->dk == 576 && a->dv == 0);
    if (!widths) return MLA_ERR_UNSUPPORTED;
    if (!(a->logit_softcap >= 0.f)) return MLA_ERR_UNSUPPORTED;
    if (a->n_seq == 0) return 0;
    if (!a->q || !a->block_table || !a->seq_lens) return MLA_ERR_NULL;
    if (a->n_pages < 1 || a->bt_stride < 1) return MLA_ERR_BAD_SHAPE;
    // rows, units of work and workgroups are counted in 31 bits
    const int64_t lim = (int64_t) 1 << 31;
    if (a->bt_stride * PAGE >= lim || (int64_t) a->n_seq * a->n_head >= (1 << 24) || (int64_t) a->n_seq * a->n_head_kv > 65535 || (int64_t) a->n_seq * a->n_head * a->bt_stride >= lim)
        return MLA_ERR_BAD_SHAPE;
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
    p.k = (const char *) a->k.data; p.k_page = a->k.nb_page; p.k_head = a->k.nb_head; p.k_row = (int) a->k.nb_row;
    p.v = (const char *) a->v.data; p.v_page = a->v.nb_page; p.v_head = a->v.nb_head; p.v_row = (int) a->v.nb_row;
    p.n_pages = a->n_pages; p.block_table = a->block_table; p.bt_stride = a->bt_stride; p.seq_lens = a->seq_lens;
    p.mask = (const char *) a->mask; p.mask_nb1 = a->mask_nb1; p.mask_ne0 = a->mask_ne0;
    p.weights = a->weights; p.w_nb1 = a->w_nb1; p.w_nb2 = a->w_nb2;
    p.dst = (char *) a->dst; p.d_nb1 = a->d_nb1; p.d_nb2 = a->d_nb2; p.dst_f32 = a->dst_type == MLA_TYPE_F32;
    p.scale_log2 = a->scale * LOG2E;
    p.cap_in  = a->logit_softcap > 0.f ? 2.f * LOG2E * a->scale / a->logit_softcap : 0.f;
    p.cap_out = a->logit_softcap * LOG2E;
    p.window = a->window; p.n_seq = a->n_seq; p.n_head = a->n_head; p.n_head_kv = a->n_head_kv; p.group = a->n_head / a->n_head_kv;
    p.row_blocks = pl.row_blocks; p.head_blocks = a->n_head_kv * pl.row_blocks; p.dv = a->dv; p.n_wg = pl.n_wg;
    p.part_o = (float *) ws; p.part_ml = (float2 *) (ws + pl.off_ml); p.items = (int2 *) (ws + pl.off_items);
    p.scores = a->weights ? (float *) (ws + pl.off_scores) : nullptr; p.lse = a->weights ? (float2 *) (ws + pl.off_lse) : nullptr;
    p.cap = a->bt_stride * PAGE;
    return (int) (a->kv_type == MLA_TYPE_F16 ? launch_all<true>(p, pl, a->dk, (hipStream_t) stream) : launch_all<false>(p, pl, a->dk, (hipStream_t) stream));
}
