// Attention of many query rows over the same keys (include/gqa_batch.h), for gfx950.
//
//   o[r] = sum_i p_i v_i,  p = softmax_i(scale * q[r] . k_i [soft cap] [+ mask]),  r = (token, head) of a group, i the rows that r sees
//
// A workgroup of four waves takes a block of query rows; tiles of keys and values come to LDS by direct loads (16 bytes a lane, no registers), the
// next ones while this one is worked on, swizzled so that both ways of reading them are free of bank conflicts.  Per tile and wave:
//   * S^T = K Q^T by 32x32x16 MFMAs: a lane holds 16 scores of one query row a block of 32 keys, the other half of the wave the other 16.  Maximum and sum of
//     a row are a lane's own business (and one exchange between the halves when the reference moves).
//   * O^T += V^T P^T: the scores' registers, exponentiated and packed, are the second operand as they are (contraction index e of half g: key 4 g + e,
//     then 8 + 4 g + e); V^T comes from LDS by transposing reads.  A lane's accumulators all belong to its query row: no rescaling across lanes.
//   * the reference of a row moves only when a score passes it by 2^8 (f16: 2^4, with P up to 2^15, so that what f16 loses of a weight is 2^-11 of it down to
//     2^-25 of the largest).
//
// Work: where there are blocks enough, a workgroup each, the heavy ones first.  Else blocks in the order (group, KV head, block) have weights (keys they see, closed
// sums), and the workgroups take equal runs of the total weight, cut at tiles.  A run that covers a block writes its result; the others leave (o, m, l)
// for gqa_batch_join_kernel.  All of that is decided from the lengths on the device: a captured launch stays valid while they change.
//
// What bounds it: the matrix units and the vector work between their products, one after the other (a tile of 64 keys of heads of 128: 32 MFMAs of 32 cycles a wave, and 32
// exponentials of 16 cycles with some 90 other instructions of 4; of heads of 64: as much vector work to half the MFMAs).  Though two or three waves share a SIMD, the cycles that either
// keeps busy add up to all there are: heads of 128 50 + 50 %, of 64 34 + 68 % (instructions counted, times their cycles); if they overlapped, heads of 64 would reach 0.95 PFLOP/s.  Prompts of 4 x 4096 tokens, 32 heads on 8,
// bf16, TFLOP/s without anything / with a mask / with a soft cap: heads of 64 596 / 477 / 388 (twice the exponentials a product), 128 909 / 775 / 669, 192 875 / 662 /
// 613, 256 594 / 437 / 466 (one wave a SIMD: 512 registers, and 28 to 46 moves between its halves a tile beside the score products); f16 of 64 667.  One prompt of 16384 tokens,
// heads of 128: 2.1 to 2.3 ms box to box, 0.96 to 1.04 PFLOP/s, where an 8192 x 8192 x 8192 library product reaches 1.20, at a clock of 1.9 to 2.0 GHz; LDS has no bank conflicts.  Fewer rows than 128 a block are bound by what a
// run waits for: 8 tokens behind 4000 rows 18 us here and 5 in the join, of which 3.2 would be the bytes.
#pragma once

#include <limits.h>

#include <type_traits>

#include "gqa_batch.hpp"

namespace mla {
namespace gqa {
namespace {

// The kernel's arguments where they lie: read again wherever `fresh` has been, which keeps those that the loop over tiles does not need out of its scalar registers.
typedef const __attribute__((address_space(4))) BatchP Params;
__device__ __forceinline__ Params * fresh() {
    Params * p = (Params *) __builtin_amdgcn_kernarg_segment_ptr();
    asm volatile("" : "+s"(p));
    return p;
}
__device__ __forceinline__ int uni(int v) { return __builtin_amdgcn_readfirstlane(v); }
__device__ __forceinline__ uint64_t uni64(uint64_t v) {
    return (uint64_t) (unsigned) __builtin_amdgcn_readfirstlane((int) (v >> 32)) << 32 | (unsigned) __builtin_amdgcn_readfirstlane((int) v);
}

// N times 64 lanes, 16 bytes each: from base + off[j] (a lane's own) plus the instruction's offset to LDS at `lds` + 1024 j, lane by lane.  Waited for by dma_wait().
template <int N> __device__ __forceinline__ void dma_tile(uint64_t base, const unsigned (&off)[N], unsigned lds) {
    constexpr int AT = N % 4;
    if constexpr (AT == 1) asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %2, %1" : : "s"(lds), "s"(base), "v"(off[0]) : "memory", "m0");
    if constexpr (AT == 2)
        asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %2, %1\n\tglobal_load_lds_dwordx4 %3, %1 offset:1024"
                     : : "s"(lds), "s"(base), "v"(off[0]), "v"(off[1]) : "memory", "m0");
    if constexpr (AT == 3)
        asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %2, %1\n\tglobal_load_lds_dwordx4 %3, %1 offset:1024\n\tglobal_load_lds_dwordx4 %4, %1 offset:2048"
                     : : "s"(lds), "s"(base), "v"(off[0]), "v"(off[1]), "v"(off[2]) : "memory", "m0");
#pragma unroll
    for (int j = AT; j < N; j += 4)
        asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %2, %1\n\tglobal_load_lds_dwordx4 %3, %1 offset:1024\n\t"
                     "global_load_lds_dwordx4 %4, %1 offset:2048\n\tglobal_load_lds_dwordx4 %5, %1 offset:3072"
                     : : "s"(lds + j * 1024), "s"(base), "v"(off[j]), "v"(off[j + 1]), "v"(off[j + 2]), "v"(off[j + 3]) : "memory", "m0");
}
template <int LEFT> __device__ __forceinline__ void dma_wait() { __builtin_amdgcn_s_waitcnt((LEFT & 15) | 0x0f70 | (LEFT >> 4) << 14); }     // all but the last LEFT loads

// Place of 16-byte chunk c of row r in a tile of rows of D values: c ^ swizzle(r).  Rows 0 .. 15 of a chunk (the reads of K), and the 64 bytes that each of
// four neighbouring rows gives to a transposing read of V, lie in banks of their own.
template <int D> __device__ __forceinline__ int swizzle(int r) {
    return D % 128 == 0 ? ((r & 3) << 2) | ((r >> 2) & 3) : ((r & 2) << 1) | ((r >> 2) & 3);
}

struct Group { int q0, nq, len; int64_t row0; };
__device__ __forceinline__ Group group_of(Params & p, int g) {
    Group r;
    r.q0 = p.q_starts ? min(max(p.q_starts[g], 0), p.n_tok) : g * p.per;
    r.nq = p.q_starts ? min(max(p.q_starts[g + 1], r.q0), p.n_tok) - r.q0 : p.per;
    r.row0 = 0;
    int most = p.cap;
    if (p.kv_starts) {
        const int at = p.kv_starts[g];
        most = at < 0 || at > p.cap ? 0 : p.cap - at;
        r.row0 = most ? at : 0;
    }
    r.len = min(max(p.lens ? p.lens[g] : p.kv_starts ? p.kv_starts[g + 1] - p.kv_starts[g] : p.cap, 0), most);
    return r;
}
// What token j of the group sees: rows [first, last).
struct Span { int first, last; };
__device__ __forceinline__ Span span_of(Params & p, const Group & g, int j) {
    const int end = p.causal ? min(max(g.len - g.nq + j + 1, 0), g.len) : p.own_lens ? min(max(p.own_lens[g.q0 + j], 0), g.len) : g.len;
    return Span{ p.window > 0 ? max(end - p.window, 0) : 0, min(end, p.mask_len) };
}
template <int BM> __device__ __forceinline__ int blocks_of(Params & p, const Group & g) { return (int) (((int64_t) g.nq * p.group + BM - 1) / BM); }
// Row / heads of a KV head's group (the quotient is off by 2^-52 of itself, and half a step from the next number).
__device__ __forceinline__ int token_of(Params & p, int row) { return (int) (((double) row + 0.5) * p.per_head); }
// The tiles that some row of block j sees: [first, last).
template <int BM, int TK> __device__ __forceinline__ Span tiles_of(Params & p, const Group & g, int j) {
    if (p.own_lens) return Span{ 0, (min(g.len, p.mask_len) + TK - 1) / TK };     // (some sequence's whole prefix)
    const int64_t rows = (int64_t) g.nq * p.group, r0 = (int64_t) j * BM;
    const int lo = p.window > 0 ? span_of(p, g, token_of(p, (int) r0)).first : 0, hi = span_of(p, g, p.causal ? token_of(p, (int) ((r0 + BM < rows ? r0 + BM : rows) - 1)) : 0).last;
    return hi > lo ? Span{ lo / TK, (hi + TK - 1) / TK } : Span{ 0, 0 };
}

// ---- the deal, in 64-bit floating point (whole numbers below 2^53), the same in all workgroups
// sum over i < n of a + i s, each held to [0, top]
__device__ __forceinline__ double sum_clamped(double a, double s, double per_s, double top, double n) {
    const double i0 = fmin(n, fmax(0., ceil(-a * per_s))), i1 = fmin(n, fmax(0., ceil((top - a) * per_s))), mid = i1 - i0;
    return mid * a + s * ((i0 + i1 - 1.) * mid * 0.5) + (n - i1) * top;
}
// Weight of blocks 0 .. n - 1 of a group: the keys each sees, times the heads of the KV head's group, and 128 keys for what a block costs by itself.
template <int BM> __device__ __forceinline__ double weight_before(Params & p, const Group & g, double n) {
    const double G = p.group, all = G * g.len, base = G * (g.len - g.nq);
    double keys;
    if (p.causal) {
        keys = sum_clamped(base + BM, BM, 1. / BM, all, n);
        if (p.window > 0) keys -= sum_clamped(base + G * (1. - p.window), BM, 1. / BM, all, n);
    } else keys = n * (p.window > 0 ? fmin(all, G * p.window) : all);
    return keys + n * G * 128.;
}
struct Pos { int g, kvh, j, tile; };             // tile: counted from the block's first
__device__ __forceinline__ bool same_item(const Pos & a, const Pos & b) { return a.g == b.g && a.kvh == b.kvh && a.j == b.j; }
// Every wave works it out for itself, a group a lane.
template <int BM, int TK> struct Deal {
    Params & p;
    const int lane;
    Group  g;                                    // this lane's
    double w, incl;                              // its weight over all KV heads, and with those of the groups before it in these 64
    // the last block that place() found: weights before it and its own, its tiles
    double before, mine;
    int    nt;
    __device__ __forceinline__ void fetch(int g0) {
        w = 0.;
        g = Group{ 0, 0, 0, 0 };
        if (g0 + lane < p.n_grp) {
            g = group_of(p, g0 + lane);
            w = weight_before<BM>(p, g, blocks_of<BM>(p, g)) * p.n_head_kv;
        }
        incl = w;
        if (p.n_grp > 1)
#pragma unroll
            for (int d = 1; d < 64; d <<= 1) { const double o = __shfl_up(incl, d, 64); if (lane >= d) incl += o; }
    }
    // the weight of all blocks; of the heaviest (the last of a group, at most) and of the heaviest among the first ones of the groups, which are the last to be begun
    __device__ __forceinline__ double total(float & most, float & late) {
        double all = 0.;
        most = late = 0.f;
        for (int g0 = 0; g0 < p.n_grp; g0 += 64) {
            fetch(g0);
            all += __shfl(incl, p.n_grp > 1 ? 63 : 0, 64);
            if (p.deal != EITHER) continue;
            const int nb = w > 0. ? blocks_of<BM>(p, g) : 0;
            float last = nb ? (float) (weight_before<BM>(p, g, nb) - weight_before<BM>(p, g, nb - 1)) : 0.f, first = nb ? (float) weight_before<BM>(p, g, 1) : 0.f;
#pragma unroll
            for (int d = 1; d < 64; d <<= 1) { last = fmaxf(last, __shfl_xor(last, d, 64)); first = fmaxf(first, __shfl_xor(first, d, 64)); }
            most = fmaxf(most, last); late = fmaxf(late, first);
        }
        return all;
    }
    __device__ __forceinline__ int tile_at(double at) const { return uni(max(min((int) ((at - before) * nt / mine), nt - 1), 0)); }
    __device__ __forceinline__ Pos place(double at) {            // after total()
        double ahead = 0.;
        for (int g0 = 0; g0 < p.n_grp; g0 += 64) {
            if (p.n_grp > 64) fetch(g0);
            const uint64_t past = __ballot(at < ahead + incl);
            if (past) {
                const int l = p.n_grp > 1 ? uni(__ffsll((unsigned long long) past) - 1) : 0;
                const Group o{ __builtin_amdgcn_readlane(g.q0, l), __builtin_amdgcn_readlane(g.nq, l), __builtin_amdgcn_readlane(g.len, l), 0 };
                const int    nb = blocks_of<BM>(p, o);
                const double per = weight_before<BM>(p, o, nb);
                before = ahead + __shfl(incl - w, l, 64);
                const int kvh = min((int) ((at - before) / per), p.n_head_kv - 1);
                before += kvh * per;
                int lo = 0, hi = nb;                              // weight_before(lo) <= at - before < weight_before(hi)
                if (!p.causal) lo = max(min((int) ((at - before) / weight_before<BM>(p, o, 1.)), nb - 1), 0);
                else
                    while (hi - lo > 1) {
                        const int mid = (lo + hi) / 2;
                        if (weight_before<BM>(p, o, mid) <= at - before) lo = mid;
                        else hi = mid;
                    }
                const double w0 = weight_before<BM>(p, o, lo);
                mine = weight_before<BM>(p, o, lo + 1.) - w0;
                before += w0;
                const Span t = tiles_of<BM, TK>(p, o, lo);
                nt = t.last - t.first;
                return Pos{ uni(g0 + l), uni(kvh), uni(lo), tile_at(at) };
            }
            ahead += __shfl(incl, p.n_grp > 1 ? 63 : 0, 64);
        }
        return Pos{ p.n_grp, 0, 0, 0 };
    }
};
// Number of block j of group g among all, an upper bound's worth apart: blocks_of(g) are at most the numbers between two groups.
template <int BM> __device__ __forceinline__ int64_t number_of(Params & p, int g, int q0) { return (int64_t) q0 * p.group / BM + g; }

// The group that a block number belongs to: the last whose first number is not past it, 64 tried at a time.
template <int BM> __device__ __forceinline__ int group_with(Params & p, int64_t id, int lane) {
    int lo = 0, n = p.n_grp;
    while (n > 1) {
        const int step = (n + 63) / 64, g = lo + lane * step;
        const bool in = lane * step < n;
        const int q0 = !in ? 0 : p.q_starts ? min(max(p.q_starts[g], 0), p.n_tok) : g * p.per;
        const int last = 63 - __clzll((long long) (__ballot(in && number_of<BM>(p, g, q0) <= id) | 1));
        n = min(step, n - last * step);
        lo += last * step;
    }
    return uni(lo);
}

__device__ __forceinline__ u32x4 lds128(unsigned at) { return *(LDS_PTR(const u32x4)) (uintptr_t) at; }
// Four rows' values of this lane's column, twice: rows r .. r + 3 and r + 8 .. r + 11 of the transposed operand.
__device__ __forceinline__ u32x4 lds_transposed(unsigned lo, unsigned hi) {
    const u32x2 a = bitcast<u32x2>(__builtin_amdgcn_ds_read_tr16_b64_v4i16((LDS_PTR(s16x4)) (uintptr_t) lo)), b = bitcast<u32x2>(__builtin_amdgcn_ds_read_tr16_b64_v4i16((LDS_PTR(s16x4)) (uintptr_t) hi));
    return u32x4{ a.x, a.y, b.x, b.y };
}
// Two numbers to 16 bits each, to nearest even, in one instruction.
typedef __attribute__((ext_vector_type(2))) float f32x2;
template <bool F16> __device__ __forceinline__ unsigned packed16(float a, float b) {
    if constexpr (F16) return bitcast<unsigned>(__builtin_convertvector(f32x2{ a, b }, f16x2));
    else               return bitcast<unsigned>(__builtin_convertvector(f32x2{ a, b }, bf16x2));
}
// An address in a register of its own, so that constants added to it become the instructions' offsets.
__device__ __forceinline__ unsigned base_of(unsigned a) { asm("" : "+v"(a)); return a; }
// scaled_score with a cap, without branches.
__device__ __forceinline__ float capped_score(float scale_log2, float cap_in, float cap_out, float a) {
    const float s = scale_log2 * a, y = fabsf(cap_in * a), u = y * y;
    const float near = fmaf(u, fmaf(u, 15.f, 420.f), 945.f), far = fast_exp2(2.f * LOG2E * y) + 1.f;
    const float r = __builtin_amdgcn_rcpf(y < 0.75f ? near : far), x = s * (fmaf(u, u + 105.f, 945.f) * r), z = copysignf(cap_out * fmaf(-2.f, r, 1.f), s);
    return y < 0.75f ? x : z;
}
// l + the two 16-bit numbers of `pair`: the sum is over the weights as they are multiplied, so that a row of one key gets its value as it is.
template <bool F16> __device__ __forceinline__ float add_pair(float l, unsigned pair) {
    if constexpr (F16) return __builtin_amdgcn_fdot2(bitcast<f16x2>(pair), f16x2{ (_Float16) 1.f, (_Float16) 1.f }, l, false);
    else               return __builtin_amdgcn_fdot2_f32_bf16(bitcast<bf16x2>(pair), bf16x2{ (__bf16) 1.f, (__bf16) 1.f }, l, false);
}
// ---- infinities and NaN among values: 0 * them must not count where a row does not see their key.  Two 16-bit numbers at a time.
template <bool F16> __device__ __forceinline__ unsigned nonfinite(unsigned x) {                // bits 15 and 31: of the halves that are
    return ((x & (F16 ? 0x7c007c00u : 0x7f807f80u)) + (F16 ? 0x04000400u : 0x00800080u)) & 0x80008000u;
}
__device__ __forceinline__ unsigned halves(unsigned bits15) { return (bits15 >> 15) * 0xffffu; }  // all bits of those halves

template <bool F16> __device__ __forceinline__ u32x2 pack4(float a, float b, float c, float d) { return u32x2{ packed16<F16>(a, b), packed16<F16>(c, d) }; }

// What is done to scores besides scaling them: a mask added, or a soft cap and perhaps a mask behind it.
enum Extra { NOTHING, MASK, CAP };

template <bool F16, int DK, int DV, int NWQ, int NWK, int TK, int NS, int OCC, Extra EXTRA>
__global__ void __launch_bounds__(64 * NWQ * NWK, OCC) gqa_batch_kernel(const BatchP) {
    constexpr int NW = NWQ * NWK, BM = 32 * NWQ, KW = TK / NWK, KB = KW / 32, KC = DK / 16, NV = DV / 32;
    constexpr int KT = TK * DK * 2, VT = TK * DV * 2, KI = KT / 1024 / NW, VI = VT / 1024 / NW;
    static_assert(KW % 32 == 0 && KI * 1024 * NW == KT && VI * 1024 * NW == VT, "whole pieces");
    // One wave a SIMD has nobody to fill its gaps: the scores' products of the next tile lie among what is done to this tile's scores.  Without / with that: 6 x 700 tokens,
    // window and cap 188 / 172 us; 4 x 4096 tokens 532 / 594 TFLOP/s, with a cap 421 / 466.  (Narrower heads: two waves a SIMD, and no registers for it.  A mask would be needed
    // for two tiles at a time.)
    constexpr bool NEXT = DK == 256 && NWK == 1 && EXTRA != MASK;
    static_assert(!NEXT || (KB == 1 && KC == 16 && NS > 2), "a score beside each product, two tiles there at a time");
    constexpr float REF = F16 ? 11.f : 0.f, SLACK = F16 ? 4.f : 8.f, MOST = F16 ? 32768.f / DK : 1024.f;
    extern __shared__ __attribute__((aligned(1024))) char lds[];
    __shared__ float2 sh_ml[NWK > 1 ? NW : 1][NWK > 1 ? 32 : 1];
    __shared__ int    sh_bad[2][NW];

    const int lane = threadIdx.x & 63, wave = uni(threadIdx.x >> 6), wq = wave % NWQ, wk = wave / NWQ, l31 = lane & 31, hh = lane >> 5;
    const unsigned lds0 = (unsigned) (uintptr_t) (LDS_PTR(char)) lds;
    Pos  at, end = { 0, 0, 0, 0 };
    int  run = blockIdx.x;
    bool single;
    {
    Params & p = *fresh();

    if (p.own_lens)                                                   // whose prefix is whose
        for (int b = blockIdx.x * 64 * NW + threadIdx.x; b < p.n_tok; b += gridDim.x * 64 * NW) {
            int lo = 0, hi = p.n_grp;                                 // q_starts[lo] <= b < q_starts[hi], where there are such
            while (hi - lo > 1) {
                const int mid = (lo + hi) / 2;
                if (p.q_starts[mid] <= b) lo = mid;
                else hi = mid;
            }
            const Group g = group_of(p, lo);
            const bool  in = b >= g.q0 && b < g.q0 + g.nq;
            p.shared[b] = in ? g.len : 0;
            p.shared_group[b] = in ? lo : -1;
        }
    // ---- this workgroup's run, or its block
    Deal<BM, TK> deal{ p, lane };
    single = p.deal == WHOLE;
    if (!single) {
        float        most, late;
        const double total = deal.total(most, late);
        const float  share = (float) total / p.n_wg;
        single = p.deal == EITHER && fmaxf(most, share + 0.5f * late) <= share + (float) JOIN_KEYS * p.group;
        if (!single) {
            const int runs = (int) fmax(total > 0. ? 1. : 0., fmin((double) p.n_wg, total / ((double) p.min_tiles * TK * p.group)));
            if ((int) blockIdx.x >= runs) {
                if ((int) blockIdx.x < p.n_wg && threadIdx.x == 0) p.tasks[blockIdx.x] = make_int4(-1, 0, 0, 0);
                return;
            }
            // (workgroups go to the eight dies in turn: neighbouring runs, which share keys, to the same one)
            const int x = blockIdx.x & 7;
            run = uni(x * (runs >> 3) + min(x, runs & 7) + (int) (blockIdx.x >> 3));
            // (the block that begins in this run and goes on in others is joined by the workgroup of this number: set where it is left)
            if (threadIdx.x == 0) p.tasks[run] = make_int4(-1, 0, 0, 0);
            auto mark = [&](int r) { return floor(total * r / runs); };
            at = deal.place(mark(run));
            if (run + 1 == runs) end.g = p.n_grp;
            else if (mark(run + 1) < deal.before + deal.mine) { end = at; end.tile = deal.tile_at(mark(run + 1)); }   // (in the same block)
            else end = deal.place(mark(run + 1));
        }
    }
    if (single) {                                                     // blocks by falling number: the later ones of a group see the more keys
        const int64_t id = (int64_t) p.blocks - 1 - blockIdx.x / p.n_head_kv;
        // (no block is left to be joined: every workgroup that the join looks at says so, those without a block among them)
        if ((int) blockIdx.x < p.n_wg && threadIdx.x == 0) p.tasks[blockIdx.x] = make_int4(-1, 0, 0, 0);
        if (id < 0) return;
        at.g = group_with<BM>(p, id, lane); at.kvh = blockIdx.x % p.n_head_kv; at.tile = 0;
        const Group g = group_of(p, at.g);
        at.j = (int) max(id - number_of<BM>(p, at.g, g.q0), (int64_t) -1);
        if (at.j < 0 || at.j >= blocks_of<BM>(p, g)) return;
    }
    }

    // ---- what does not change: a lane's places in the tiles
    // (a wave's loads of a tile lie one behind the other; an instruction's offset counts for both its places, so one that is ahead in LDS is taken back in memory)
    auto step_of = [](int per, int j) { return j < per % 4 ? j : (j - per % 4) % 4; };
    auto row_in = [&](int d, int per, int j, int lane) { return ((wave * per + j) * 64 + lane) / (d / 8); };
    auto place_in = [&](int d, int per, int j, int lane) { const int r = row_in(d, per, j, lane), c = ((wave * per + j) * 64 + lane) % (d / 8); return (c ^ (d % 128 == 0 ? swizzle<128>(r) : swizzle<64>(r))) * 16 + (4 - step_of(per, j)) * 1024; };
    int k_row, v_row;
    unsigned k_at[KI], v_at[VI];
    {
        Params & p = *fresh();
        k_row = p.k_row; v_row = p.v_row;
#pragma unroll
        for (int j = 0; j < KI; j++) k_at[j] = (unsigned) (row_in(DK, KI, j, lane) * k_row + place_in(DK, KI, j, lane));
#pragma unroll
        for (int j = 0; j < VI; j++) v_at[j] = (unsigned) (row_in(DV, VI, j, lane) * v_row + place_in(DV, VI, j, lane));
    }
    // transposing reads: row, 16-byte chunk and half of it; the addresses of a chunk of 32 columns, for rows 0 .. 3 and 8 .. 11 of 16
    const int vq = hh * 4 + ((lane >> 2) & 3), vc = ((lane >> 4) & 1) * 2 + ((lane & 3) >> 1), vsub = (lane & 1) * 8;
    // (chunks beyond those that the swizzle moves among are whole steps further on)
    constexpr int VP = DV % 128 == 0 ? 4 : 2, KP = DK % 128 == 0 ? 8 : 4;
    unsigned v_lo[VP], v_hi[VP], k_lo[KP];
#pragma unroll
    for (int n = 0; n < VP; n++) {
        v_lo[n] = vq * (DV * 2) + (((n * 4 + vc) ^ swizzle<DV>(vq)) * 16) + vsub;
        v_hi[n] = (vq + 8) * (DV * 2) + (((n * 4 + vc) ^ swizzle<DV>(vq + 8)) * 16) + vsub;
    }
#pragma unroll
    for (int c = 0; c < KP; c++) k_lo[c] = l31 * (DK * 2) + (((2 * c + hh) ^ swizzle<DK>(l31)) * 16);

    end = Pos{ uni(end.g), uni(end.kvh), uni(end.j), uni(end.tile) };
    single = uni(single);
    for (;;) {
        at = Pos{ uni(at.g), uni(at.kvh), uni(at.j), uni(at.tile) };
        Params & p = *fresh();
        if (at.g >= p.n_grp) return;
        const Group g = group_of(p, at.g);
        const int   nb = blocks_of<BM>(p, g);
        const Span  ts = nb > 0 ? tiles_of<BM, TK>(p, g, at.j) : Span{ 0, 0 };
        const int   nt = ts.last - ts.first;
        const bool  ends_here = !single && same_item(at, end);
        const int   t0 = uni(ts.first + at.tile), t1 = uni(ends_here ? ts.first + end.tile : ts.last);
        const bool  begins = at.tile == 0, whole = begins && !ends_here;
        const int   row0 = at.j * BM + wq * 32;
        const int64_t item = (number_of<BM>(p, at.g, g.q0) + at.j) * p.n_head_kv + at.kvh;
        const bool  direct = whole && !p.own_lens;
        const int64_t slot = whole ? 2 * (int64_t) p.n_wg + item : 2 * run + (begins ? 1 : 0);

        if (t0 < t1) {
            if (threadIdx.x == 0) {
                if (begins) { p.items[item].x = (int) slot; p.items[item].y = run; }
                if (!ends_here) p.items[item].z = run;
            }
            // (what the loop over tiles needs of the arguments)
            const float scale_log2 = p.scale_log2, cap_in = EXTRA == CAP ? p.cap_in : 0.f, cap_out = EXTRA == CAP ? p.cap_out : 0.f, mask_unit = EXTRA == MASK ? p.mask_unit : 0.f;
            const bool  masks = EXTRA != NOTHING && p.mask;
            // ---- this lane's query row (rows past the last repeat it)
            const int  rows = g.nq * p.group, r = min(row0 + l31, rows - 1), tok = token_of(p, r), head = at.kvh * p.group + r - tok * p.group;
            const Span s = span_of(p, g, tok);
            // the rows that all of the wave's and that any of them see, and the same of the block: spans move on with the token, but for sequences' own lengths
            const int64_t last_row = min((int64_t) (at.j + 1) * BM, (int64_t) rows) - 1;
            Span s_first, s_last, b_first, b_last;
            if (p.own_lens) {
                int lo = s.last, hi = s.last, least = s.last;
                if constexpr (BM > 32) for (int i = lane; i < BM; i += 64) least = min(least, span_of(p, g, token_of(p, (int) min((int64_t) at.j * BM + i, last_row))).last);
#pragma unroll
                for (int d = 1; d < 64; d <<= 1) { lo = min(lo, __shfl_xor(lo, d, 64)); hi = max(hi, __shfl_xor(hi, d, 64)); least = min(least, __shfl_xor(least, d, 64)); }
                s_first = Span{ 0, uni(lo) }; s_last = Span{ 0, uni(hi) }; b_first = b_last = Span{ 0, uni(least) };
            } else {
                s_first = Span{ uni(__shfl(s.first, 0, 64)), uni(__shfl(s.last, 0, 64)) }; s_last = Span{ uni(__shfl(s.first, 31, 64)), uni(__shfl(s.last, 31, 64)) };
                b_first = span_of(p, g, token_of(p, at.j * BM)); b_last = span_of(p, g, token_of(p, (int) last_row));
            }
            const int64_t seq = p.own_lens ? g.q0 : at.g;             // whose pages
            const char * mask = EXTRA != NOTHING && p.mask ? p.mask + (p.own_lens ? (int64_t) (g.q0 + tok) : at.g) * p.mask_nb1 : nullptr;

            const int64_t k_off = (int64_t) at.kvh * p.k_head + (p.block_table ? 0 : at.g * p.k_page + g.row0 * p.k_row);
            const int64_t v_off = (int64_t) at.kvh * p.v_head + (p.block_table ? 0 : at.g * p.v_page + g.row0 * p.v_row);
            const uint64_t k_base = uni64((uint64_t) (uintptr_t) p.k + (uint64_t) k_off), v_base = uni64((uint64_t) (uintptr_t) p.v + (uint64_t) v_off);
            const int32_t * pages = p.block_table + (p.block_table ? seq * p.bt_stride : 0);
            const int64_t n_pages = p.n_pages, k_page = p.block_table ? p.k_page : 0, v_page = p.block_table ? p.v_page : 0;
            const bool paged = p.block_table != nullptr;
            auto good = [&](int id) { return id >= 0 && id < n_pages; };
            // (through the scalar cache, nothing writes them meanwhile: a vector load would be waited for together with the tiles that are under way)
            auto page_at = [&](int t) { return *(const int32_t __attribute__((address_space(4))) *) (uintptr_t) (pages + t * TK / PAGE); };
            auto fetch = [&](int t, int id, int buf) {                // tile t to LDS
                const int key0 = t * TK, row = paged ? key0 % PAGE : key0, pg = good(id) ? id : 0;    // (a bad id: page 0 is read, not used)
                const uint64_t kb = uni64(k_base + (uint64_t) (pg * k_page + (int64_t) row * k_row)) - 4096, vb = uni64(v_base + (uint64_t) (pg * v_page + (int64_t) row * v_row)) - 4096;
                const unsigned to = uni(lds0 + buf * (KT + VT)), k_to = to + wave * (KI * 1024), v_to = to + KT + wave * (VI * 1024);
                if (key0 + TK <= g.len) {
                    dma_tile<KI>(kb, k_at, k_to);
                    dma_tile<VI>(vb, v_at, v_to);
                } else {                                              // (rows past the last repeat it)
                    const int last = g.len - key0 - 1, me = (int) base_of(lane);     // (worked out here, and not kept for here)
                    unsigned k_end[KI], v_end[VI];
#pragma unroll
                    for (int j = 0; j < KI; j++) k_end[j] = (unsigned) (min(row_in(DK, KI, j, me), last) * k_row + place_in(DK, KI, j, me));
#pragma unroll
                    for (int j = 0; j < VI; j++) v_end[j] = (unsigned) (min(row_in(DV, VI, j, me), last) * v_row + place_in(DV, VI, j, me));
                    dma_tile<KI>(kb, k_end, k_to);
                    dma_tile<VI>(vb, v_end, v_to);
                }
            };
            // the mask's numbers of a tile; rows past the last that the lane's query sees: -infinity
            const bool mask_whole = EXTRA != NOTHING && mask && !uni(__any(((uintptr_t) mask & 7) != 0));
            u32x2 mk[KB][4];
            auto fetch_mask = [&](int t) {
                if constexpr (EXTRA != NOTHING)
                    if (mask) {
                        const int  i0 = t * TK + wk * KW + hh * 4;
                        const bool whole_tile = mask_whole && t * TK + TK <= b_first.last;
#pragma unroll
                        for (int b = 0; b < KB; b++)
#pragma unroll
                            for (int c = 0; c < 4; c++) {
                                const int i = i0 + b * 32 + c * 8;
                                const char * src = mask + (int64_t) i * 2;
                                if (whole_tile) mk[b][c] = *(const u32x2 *) src;
                                else {
                                    unsigned short h[4];
#pragma unroll
                                    for (int e = 0; e < 4; e++) h[e] = i + e < s.last ? *(const unsigned short *) (src + 2 * e) : (unsigned short) 0xfc00;
                                    mk[b][c] = u32x2{ h[0] | ((unsigned) h[1] << 16), h[2] | ((unsigned) h[3] << 16) };
                                }
                            }
                    }
            };
            auto masked_by = [&](int b, int e) { return f16_bits_to_f32((mk[b][e >> 2][(e >> 1) & 1] >> (16 * (e & 1))) & 0xffffu); };

            u32x4 qf[KC];
            {
                const char * src = p.q + (int64_t) (g.q0 + tok) * p.q_nb2 + (int64_t) head * p.q_nb1 + hh * 16;
#pragma unroll
                for (int c = 0; c < KC; c++) {
                    qf[c] = *(const u32x4 *) (src + c * 32);
#pragma unroll
                    for (int e = 0; e < 4; e++) qf[c][e] ^= p.flip;
                }
            }
            float  m, l;
            f32x16 acc[NV];
            // Infinities and NaN among keys and values must not count where a row does not see them, and 0 * them does.  The piece is worked on as if there were none; if a result
            // is not finite, once more from the start, `safe`: with the infinities and NaN among the values of every tile that not all rows see whole noted for the rows that
            // see them, and taken for zeros, and with masked scores set and not added to.  So is a piece whose largest scores come of a large finite number of the mask: sums that
            // begin with one of size x lose up to dk / 16 half steps of it (2^-20 x for heads of 256), added last it costs a single one.  Up to `MOST` that is no more than 2^-13
            // of a score in log2 units for f16, 2^-10 for bf16: less than a fifth of what the weights' own rounding is off by.
            unsigned up[(NV + 1) / 2], down[(NV + 1) / 2];            // safe: results that a +infinity (-infinity, NaN: both) belongs to
            bool safe = false;

            // S^T of the wave's keys; a mask is where the sums begin (in units of the products)
            auto products = [&](unsigned kt, f32x16 (&sc)[KB], auto with_mask) {
                unsigned at[KP];
#pragma unroll
                for (int c = 0; c < KP; c++) at[c] = base_of(kt + k_lo[c]);
                f32x16 start[KB];
#pragma unroll
                for (int b = 0; b < KB; b++)
#pragma unroll
                    for (int e = 0; e < 16; e++) start[b][e] = 0.f;
                if constexpr (decltype(with_mask)::value)
#pragma unroll
                    for (int b = 0; b < KB; b++)
#pragma unroll
                        for (int e = 0; e < 16; e++) start[b][e] = fmaf((float) bitcast<f16x2>(mk[b][e >> 2][(e >> 1) & 1])[e & 1], mask_unit, 0.f);   // (one instruction, converting; a product alone is two)
#pragma unroll
                for (int b = 0; b < KB; b++) {
                    sc[b] = start[b];
#pragma unroll
                    for (int c = 0; c < KC; c++) sc[b] = mfma32<F16>(lds128(at[c % KP] + c / KP * KP * 32 + b * 32 * (DK * 2)), qf[c], sc[b]);
                }
                // the order of it: reads some ahead of the products
                constexpr int LEAD = KC < 8 ? KC : 8;
                __builtin_amdgcn_sched_group_barrier(0x100, LEAD, 0);
#pragma unroll
                for (int i = 0; i < KB * KC - LEAD; i++) {
                    __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
                    __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);
                }
                __builtin_amdgcn_sched_group_barrier(0x008, LEAD, 0);
            };

            f32x16 next;                                              // NEXT: the scores of the tile that comes
            // something for every score of a tile, each(0 .. KB * 16 - 1); NEXT: beside the products of the tile at kn, keys read LEAD products ahead
            auto beside = [&](unsigned kn, auto && each) {
                if constexpr (NEXT) {
                    constexpr int LEAD = 4;
                    unsigned at[KP];
                    u32x4    kf[LEAD];
#pragma unroll
                    for (int c = 0; c < KP; c++) at[c] = base_of(kn + k_lo[c]);
                    auto key = [&](int c) { return lds128(at[c % KP] + c / KP * KP * 32); };
#pragma unroll
                    for (int c = 0; c < LEAD; c++) kf[c] = key(c);
#pragma unroll
                    for (int e = 0; e < 16; e++) next[e] = 0.f;
                    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
                    for (int c = 0; c < KC; c++) {
                        next = mfma32<F16>(kf[c % LEAD], qf[c], next);
                        if (c + LEAD < KC) kf[c % LEAD] = key(c + LEAD);
                        each(c);
                        __builtin_amdgcn_sched_barrier(0);
                    }
                } else
#pragma unroll
                    for (int i = 0; i < KB * 16; i++) each(i);
            };

            for (;;) {
                m = -INFINITY; l = 0.f;
#pragma unroll
                for (int n = 0; n < NV; n++)
#pragma unroll
                    for (int e = 0; e < 16; e++) acc[n][e] = 0.f;
#pragma unroll
                for (int n = 0; n < (NV + 1) / 2; n++) up[n] = down[n] = 0;
            __syncthreads();                                          // (LDS is free of what was before)
            fetch_mask(t0);
            // (NS - 1 tiles are under way at a time; page ids are read a tile ahead of that)
            int ids[NS];
#pragma unroll
            for (int i = 0; i < NS; i++) ids[i] = paged ? page_at(min(t0 + i, t1 - 1)) : 0;
#pragma unroll
            for (int i = 0; i < NS - 1; i++) if (t0 + i < t1) fetch(t0 + i, ids[i], i);
            int buf = 0;
            if constexpr (NEXT) {
                if (t0 + NS - 2 < t1) dma_wait<(NS - 2) * (KI + VI)>();
                else                  dma_wait<0>();
                __syncthreads();
                beside(uni(lds0), [](int) {});
            }
            for (int t = t0; t < t1; t++) {
                constexpr int AHEAD = NS - 2 - NEXT;                  // tiles that need not be there yet
                if (AHEAD > 0 && t + NS - 2 < t1) dma_wait<AHEAD * (KI + VI)>();
                else                              dma_wait<0>();
                __syncthreads();
                const int  key0 = t * TK + wk * KW;
                const bool use = !paged || good(ids[0]);
                if (t + NS - 1 < t1) fetch(t + NS - 1, ids[NS - 1], buf == 0 ? NS - 1 : buf - 1);
#pragma unroll
                for (int i = 0; i + 1 < NS; i++) ids[i] = ids[i + 1];
                if (paged && t + NS < t1) ids[NS - 1] = page_at(t + NS);
                const unsigned kn = uni(lds0 + (buf + 1 == NS ? 0 : buf + 1) * (KT + VT));                                   // (behind the last tile: what was there)
                const unsigned kt = uni(lds0 + buf * (KT + VT) + wk * KW * (DK * 2)), vt = uni(lds0 + buf * (KT + VT) + KT + wk * KW * (DV * 2));
                if (safe && ((EXTRA != NOTHING && masks) || t * TK < b_last.first || t * TK + TK > b_first.last)) {
                    unsigned bad = 0;
                    const unsigned mine = lds0 + buf * (KT + VT) + KT + threadIdx.x * 16;
#pragma unroll
                    for (int i = 0; i < VI; i++) {
                        const u32x4 x = lds128(mine + i * NW * 1024);
                        bad |= nonfinite<F16>(x.x) | nonfinite<F16>(x.y) | nonfinite<F16>(x.z) | nonfinite<F16>(x.w);
                    }
                    const int found = __any(bad != 0);
                    if (lane == 0) sh_bad[t & 1][wave] = found;
                    __syncthreads();
                    int any = 0;
#pragma unroll
                    for (int w = 0; w < NW; w++) any |= sh_bad[t & 1][w];
                    if (uni(any)) {
#pragma unroll 1
                        for (int n = 0; n < NV; n++) {
                            unsigned u = 0, d = 0;
#pragma unroll 1
                            for (int i = 0; i < KW; i++) {
                                const int key = key0 + i;
                                bool sees = use && key >= s.first && key < s.last;
                                if constexpr (EXTRA != NOTHING) if (mask && sees) sees = *(const unsigned short *) (mask + (int64_t) key * 2) != 0xfc00;
#pragma unroll
                                for (int c = 0; c < 4; c++) {
                                    const u32x2 x = *(LDS_PTR(const u32x2)) (uintptr_t) (vt + i * (DV * 2) + (((n * 4 + c) ^ swizzle<DV>(i)) * 16) + hh * 8);
#pragma unroll
                                    for (int e = 0; e < 4; e++) {
                                        const float f = from16<F16>((unsigned short) (x[e >> 1] >> (16 * (e & 1))));
                                        if (sees && !(f < INFINITY)) u |= 1u << (4 * c + e);                    // infinity or NaN
                                        if (sees && !(f > -INFINITY)) d |= 1u << (4 * c + e);
                                    }
                                }
                            }
#pragma unroll
                            for (int k = 0; k < (NV + 1) / 2; k++) if (k == n / 2) { up[k] |= u << (n & 1) * 16; down[k] |= d << (n & 1) * 16; }
                        }
                        __syncthreads();
#pragma unroll
                        for (int i = 0; i < VI; i++) {
                            u32x4 x = lds128(mine + i * NW * 1024);
#pragma unroll
                            for (int e = 0; e < 4; e++) x[e] &= ~halves(nonfinite<F16>(x[e]));
                            *(LDS_PTR(u32x4)) (uintptr_t) (mine + i * NW * 1024) = x;
                        }
                        __syncthreads();
                    }
                }
                if (use && key0 < s_last.last && key0 + KW > s_first.first) {
                    f32x16 sc[KB];
                    u32x4  pf[KB][2];
                    if constexpr (NEXT)              sc[0] = next;
                    else if (EXTRA == MASK && !safe) products(kt, sc, std::bool_constant<EXTRA == MASK>());
                    else                             products(kt, sc, std::false_type());
                    float top, unit = scale_log2;                   // what makes log2 units of sc
                    const bool all = key0 + KW <= s_first.last && key0 >= s_last.first;
                    if (EXTRA != CAP && all && !(EXTRA == MASK && safe)) {
                        top = sc[0][0];
                        beside(kn, [&](int i) { top = fmaxf(top, sc[i >> 4][i & 15]); });
                        top *= unit;
                    } else {
                        top = -INFINITY;
                        // a soft cap far above the scores of this tile: tanh(y) / y by its series to y^10, off by 2^-31 where |y| < 1/4
                        bool small = false;
                        if constexpr (EXTRA == CAP) {
                            float most = 0.f;
#pragma unroll
                            for (int b = 0; b < KB; b++)
#pragma unroll
                                for (int e = 0; e < 16; e++) most = fmaxf(most, fabsf(sc[b][e]));
                            small = cap_out != 0.f && !uni(__any(!(most * cap_in < 0.25f)));
                        }
                        // (a pass over the scores for each thing that is done to them, none with a branch in it)
                        if (EXTRA == CAP && small)
                            beside(kn, [&](int i) {
                                const float x = sc[i >> 4][i & 15], y = cap_in * x, u = y * y;
                                sc[i >> 4][i & 15] = x * (scale_log2 * fmaf(u, fmaf(u, fmaf(u, fmaf(u, fmaf(u, -1382.f / 155925, 62.f / 2835), -17.f / 315), 2.f / 15), -1.f / 3), 1.f));
                            });
                        else if (EXTRA == CAP && cap_out != 0.f) beside(kn, [&](int i) { sc[i >> 4][i & 15] = capped_score(scale_log2, cap_in, cap_out, sc[i >> 4][i & 15]); });
                        else beside(kn, [&](int i) { sc[i >> 4][i & 15] *= scale_log2; });
                        if (EXTRA == CAP ? mask != nullptr : EXTRA == MASK && safe)
#pragma unroll
                            for (int b = 0; b < KB; b++)
#pragma unroll
                                for (int e = 0; e < 16; e++) {
                                    const float f = masked_by(b, e), v = fmaf(f, LOG2E, sc[b][e]);
                                    sc[b][e] = f == -INFINITY ? -INFINITY : v;
                                }
                        if (!all) {
                            const int from = s.first - key0 - hh * 4;
                            const unsigned n = max(s.last - s.first, 0);
#pragma unroll
                            for (int b = 0; b < KB; b++)
#pragma unroll
                                for (int e = 0; e < 16; e++) sc[b][e] = (unsigned) (b * 32 + (e >> 2) * 8 + (e & 3) - from) < n ? sc[b][e] : -INFINITY;
                        }
#pragma unroll
                        for (int b = 0; b < KB; b++)
#pragma unroll
                            for (int e = 0; e < 16; e++) top = fmaxf(top, sc[b][e]);
                        unit = 1.f;
                    }
                    if (EXTRA != NOTHING && t + 1 < t1) fetch_mask(t + 1);
                    if (__any(top > m + (REF + SLACK))) {             // the reference moves
                        top = fmaxf(top, xor32(top));
                        const float nm = fmaxf(top - REF, m);
                        const float a  = m == nm ? 1.f : fast_exp2(m - nm);
                        m = nm;
                        l *= a;
#pragma unroll
                        for (int n = 0; n < NV; n++)
#pragma unroll
                            for (int e = 0; e < 16; e++) acc[n][e] *= a;
                    }
                    const float mm = m == -INFINITY ? 0.f : m;
                    // O^T += V^T P^T, 32 columns and 16 keys a product, in the order as it stands here: values are read LEAD products ahead, and between the products
                    // of 16 keys lie the weights of the next 16 (a pair's exponentials in one place, its rounding and sum in the next).
                    constexpr int LEAD = NV < 4 ? NV : 4, ALL = KB * 2 * NV, PAIRS = KB * 8;
                    unsigned lo[VP], hi[VP];
#pragma unroll
                    for (int n = 0; n < VP; n++) { lo[n] = base_of(vt + v_lo[n]); hi[n] = base_of(vt + v_hi[n]); }
                    auto value = [&](int i) { const int off = i / NV * 16 * (DV * 2) + i % NV / VP * VP * 64; return lds_transposed(lo[i % VP] + off, hi[i % VP] + off); };
                    float  e0 = 0.f, e1 = 0.f;
                    auto power = [&](int i) {                         // pair i: keys 2 i, 2 i + 1 of the lane's
                        if (i > 0 && i <= PAIRS) {
                            const unsigned h = packed16<F16>(e0, e1);
                            l = add_pair<F16>(l, h);
                            pf[(i - 1) >> 3][((i - 1) >> 2) & 1][(i - 1) & 3] = h;
                        }
                        if (i < PAIRS) {
                            e0 = fast_exp2(fmaf(sc[i >> 3][(2 * i) & 15], unit, -mm));
                            e1 = fast_exp2(fmaf(sc[i >> 3][(2 * i + 1) & 15], unit, -mm));
                        }
                    };
                    u32x4 vf[LEAD];
#pragma unroll
                    for (int i = 0; i < LEAD; i++) vf[i] = value(i);
                    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
                    for (int i = 0; i < 5; i++) power(i);
                    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
                    for (int i = 0; i < ALL; i++) {
                        acc[i % NV] = mfma32<F16>(vf[i % LEAD], pf[i / NV >> 1][i / NV & 1], acc[i % NV]);
                        if (i + LEAD < ALL) vf[i % LEAD] = value(i + LEAD);
                        if (NV <= 4) {
#pragma unroll
                            for (int k = 0; k < 4 / (NV < 4 ? NV : 4); k++) power(5 + i * (4 / (NV < 4 ? NV : 4)) + k);
                        } else if (i % (NV / 4) == 0) power(5 + i / (NV / 4));
                        __builtin_amdgcn_sched_barrier(0);
                    }
                }
                else {
                    if (EXTRA != NOTHING && t + 1 < t1) fetch_mask(t + 1);
                    if constexpr (NEXT) beside(kn, [](int) {});
                }
                buf = buf + 1 == NS ? 0 : buf + 1;
            }
                if (safe) break;
                float odd = l * 0.f;                                  // NaN if anything is not finite
                if (EXTRA == MASK && fabsf(m + REF) > MOST - SLACK && m != -INFINITY) odd = NAN;
#pragma unroll
                for (int n = 0; n < NV; n++)
#pragma unroll
                    for (int e = 0; e < 16; e++) odd = fmaf(acc[n][e], 0.f, odd);
                const int found = __any(!(odd == 0.f));
                if (lane == 0) sh_bad[0][wave] = found;
                __syncthreads();
                int any = 0;
#pragma unroll
                for (int w = 0; w < NW; w++) any |= sh_bad[0][w];
                if (!uni(any)) break;
                safe = true;
            }
            bool noted = false;
#pragma unroll
            for (int n = 0; n < (NV + 1) / 2; n++) noted = noted || (up[n] | down[n]) != 0;
            if (__any(noted)) {
#pragma unroll
                for (int n = 0; n < NV; n++)
#pragma unroll
                    for (int e = 0; e < 16; e++) {
                        const unsigned bit = 1u << ((n & 1) * 16 + e);
                        if (up[n / 2] & bit) acc[n][e] += INFINITY;
                        if (down[n / 2] & bit) acc[n][e] -= INFINITY;
                    }
            }
            l += xor32(l);

            if constexpr (NWK > 1) {                                  // the waves that took other keys of the same rows
                if (hh == 0) sh_ml[wave][l31] = make_float2(m, l);
                __syncthreads();
                float M = -INFINITY, L = 0.f;
#pragma unroll
                for (int w = 0; w < NWK; w++) M = fmaxf(M, sh_ml[w * NWQ + wq][l31].x);
#pragma unroll
                for (int w = 0; w < NWK; w++) { const float2 ml = sh_ml[w * NWQ + wq][l31]; L += ml.y == 0.f ? 0.f : ml.y * fast_exp2(ml.x - M); }
                const float f = l == 0.f ? 0.f : fast_exp2(m - M);
                f32x4 * box = (f32x4 *) lds + (size_t) (wave - NWQ) * NV * 4 * 64 + lane;
                if (wk > 0) {
#pragma unroll
                    for (int n = 0; n < NV; n++)
#pragma unroll
                        for (int c = 0; c < 4; c++) box[(n * 4 + c) * 64] = f32x4{ acc[n][4 * c], acc[n][4 * c + 1], acc[n][4 * c + 2], acc[n][4 * c + 3] } * f;
                }
                __syncthreads();
                if (wk == 0) {
#pragma unroll
                    for (int n = 0; n < NV; n++)
#pragma unroll
                        for (int c = 0; c < 4; c++) {
                            f32x4 o = f32x4{ acc[n][4 * c], acc[n][4 * c + 1], acc[n][4 * c + 2], acc[n][4 * c + 3] } * f;
#pragma unroll
                            for (int w = 1; w < NWK; w++) o += ((const f32x4 *) lds)[(size_t) ((w - 1) * NWQ + wq) * NV * 4 * 64 + (n * 4 + c) * 64 + lane];
#pragma unroll
                            for (int e = 0; e < 4; e++) acc[n][4 * c + e] = o[e];
                        }
                }
                m = M; l = L;
            }
            if (wk == 0) {
                if (direct) {
                    const float inv = l == 0.f ? 0.f : 1.f / l;       // (a NaN stays one)
                    char * dst = p.dst + (int64_t) (g.q0 + tok) * p.d_nb2 + (int64_t) head * p.d_nb1 + hh * 8;
                    if (row0 + l31 < rows)
#pragma unroll
                        for (int n = 0; n < NV; n++)
#pragma unroll
                            for (int c = 0; c < 4; c++)
                                *(u32x2 *) (dst + n * 64 + c * 16) = pack4<F16>(acc[n][4 * c] * inv, acc[n][4 * c + 1] * inv, acc[n][4 * c + 2] * inv, acc[n][4 * c + 3] * inv);
                } else {
                    f32x4 * to = (f32x4 *) p.part_o + slot * (BM * DV / 4) + wq * 64 + lane;
#pragma unroll
                    for (int n = 0; n < NV; n++)
#pragma unroll
                        for (int c = 0; c < 4; c++) to[(n * 4 + c) * NWQ * 64] = f32x4{ acc[n][4 * c], acc[n][4 * c + 1], acc[n][4 * c + 2], acc[n][4 * c + 3] };
                    if (hh == 0) p.part_ml[slot * BM + wq * 32 + l31] = make_float2(m, l);
                }
            }
            if (begins && ends_here && threadIdx.x == 0) p.tasks[run] = make_int4((int) item, g.q0, rows, at.j);
        } else if (nt == 0) {                                         // no row of this block sees a key (several workgroups may find so)
            for (int i = threadIdx.x; i < BM * (DV / 4) && !p.own_lens; i += 64 * NW) {
                const int64_t r = (int64_t) at.j * BM + i / (DV / 4);
                if (r >= (int64_t) g.nq * p.group) break;
                const int tok = (int) (r / p.group), head = at.kvh * p.group + (int) (r - (int64_t) tok * p.group);
                *(u32x2 *) (p.dst + (int64_t) (g.q0 + tok) * p.d_nb2 + (int64_t) head * p.d_nb1 + i % (DV / 4) * 8) = u32x2{ 0u, 0u };
            }
        } else if (ends_here && at.tile > 0) {                        // nothing of a block that others share: an empty piece
            for (int i = threadIdx.x; i < BM; i += 64 * NW) p.part_ml[slot * BM + i] = make_float2(-INFINITY, 0.f);
        }
        if (ends_here || single) return;
        at.tile = 0;
        if (++at.j >= nb) {
            at.j = 0;
            if (++at.kvh == p.n_head_kv) {
                at.kvh = 0;
                do at.g++; while (at.g < p.n_grp && blocks_of<BM>(p, group_of(p, at.g)) == 0);
            }
        }
    }
}

// Joins the pieces of one block: o = sum_i o_i 2^(m_i - M) / sum_i l_i 2^(m_i - M).  Grid: x = runs, each of which may leave one block that goes on in others, y = 32 columns of
// the result.  A thread takes 16 columns of its row (4 loads a piece) and, where a block has fewer than 128 rows, every second or fourth piece.  Its three dependent loads (task, item,
// pieces) bound it where pieces are few: 4.3 us when nothing is to be joined, 5.3 for 8 tokens behind 4000 rows; 12 for 8 x 512 tokens behind 5000 to 16384 rows (768 runs).
template <bool F16, int DV, int NWQ>
__global__ void __launch_bounds__(256) gqa_batch_join_kernel(const BatchP p) {
    constexpr int BM = 32 * NWQ, PG = 4 / NWQ, AHEAD = 4;
    __shared__ float2 sh_ml[PG > 1 ? PG - 1 : 1][PG > 1 ? BM * 2 : 1];
    __shared__ f32x4  sh_o[PG > 1 ? PG - 1 : 1][4][PG > 1 ? BM * 2 : 1];
    const int4 task = p.tasks[blockIdx.x];                            // item, first token of the group, its rows, block
    if (task.x < 0) return;
    const int4 it = p.items[task.x];                                  // slot of the first piece, first and last run
    const int lane = threadIdx.x & 63, wq = (threadIdx.x >> 6) % NWQ, pg = (threadIdx.x >> 6) / NWQ, row = wq * 32 + (lane & 31), mine = wq * 64 + lane;
    const int pieces = it.z - it.y + 1;
    auto slot = [&](int i) -> int64_t { return i ? 2 * (it.y + (int64_t) i) : it.x; };
    float M = -INFINITY, L = 0.f;
    f32x4 o[4] = {};
    for (int i0 = pg; i0 < pieces; i0 += PG * AHEAD) {                // (pieces past the last repeat it, without weight)
        float2 ml[AHEAD];
        f32x4  x[AHEAD][4];
#pragma unroll
        for (int a = 0; a < AHEAD; a++) {
            const int64_t s = slot(min(i0 + a * PG, pieces - 1));
            ml[a] = p.part_ml[s * BM + row];
#pragma unroll
            for (int c = 0; c < 4; c++) x[a][c] = ((const f32x4 *) p.part_o)[s * (BM * DV / 4) + ((int) blockIdx.y * 4 + c) * NWQ * 64 + mine];
        }
        float top = M;
#pragma unroll
        for (int a = 0; a < AHEAD; a++) if (ml[a].y != 0.f) top = fmaxf(top, ml[a].x);
        const float f = M == top ? 1.f : fast_exp2(M - top);
        L *= f; M = top;
#pragma unroll
        for (int c = 0; c < 4; c++) o[c] *= f;
#pragma unroll
        for (int a = 0; a < AHEAD; a++) {
            if (ml[a].y == 0.f || i0 + a * PG >= pieces) continue;    // (an empty piece has no sums)
            const float w = fast_exp2(ml[a].x - top);
            L += ml[a].y * w;
#pragma unroll
            for (int c = 0; c < 4; c++) o[c] += x[a][c] * w;
        }
    }
    if constexpr (PG > 1) {
        if (pg) {
            sh_ml[pg - 1][mine] = make_float2(M, L);
#pragma unroll
            for (int c = 0; c < 4; c++) sh_o[pg - 1][c][mine] = o[c];
        }
        __syncthreads();
        if (pg) return;
#pragma unroll
        for (int q = 0; q < PG - 1; q++) {
            const float2 ml = sh_ml[q][mine];
            if (ml.y == 0.f) continue;
            const float top = fmaxf(M, ml.x), f = M == top ? 1.f : fast_exp2(M - top), w = fast_exp2(ml.x - top);
            L = L * f + ml.y * w; M = top;
#pragma unroll
            for (int c = 0; c < 4; c++) o[c] = o[c] * f + sh_o[q][c][mine] * w;
        }
    }
    const int r = task.w * BM + row;
    if (r >= task.z) return;
    const int tok = r / p.group, head = task.x % p.n_head_kv * p.group + r - tok * p.group;
    const float inv = L == 0.f ? 0.f : 1.f / L;                       // (a NaN stays one)
    char * dst = p.dst + (int64_t) (task.y + tok) * p.d_nb2 + (int64_t) head * p.d_nb1 + ((int) blockIdx.y * 32 + (lane >> 5) * 4) * 2;
#pragma unroll
    for (int c = 0; c < 4; c++) *(u32x2 *) (dst + c * 16) = pack4<F16>(o[c].x * inv, o[c].y * inv, o[c].z * inv, o[c].w * inv);
}

// ---------------------------------------------------------------- host

template <bool F16, int DK, int DV, int NWQ, int NWK, int TK, int NS, int OCC, Extra EXTRA>
hipError_t launch_batch(const BatchP & p, const BatchPlan & pl, hipStream_t st) {
    constexpr int lds = NS * TK * (DK + DV) * 2;
    static_assert(OCC * (lds + NWQ * NWK * 8 + (NWK > 1 ? NWQ * NWK * 32 * 8 : 0)) <= 160 * 1024, "LDS");
    static std::atomic<uint64_t> granted{ 0 };
    hipError_t e = grant_lds(gqa_batch_kernel<F16, DK, DV, NWQ, NWK, TK, NS, OCC, EXTRA>, lds, granted);
    if (e != hipSuccess) return e;
    const int64_t grid = p.deal == RUNS ? p.n_wg : (int64_t) p.blocks * p.n_head_kv;
    hipLaunchKernelGGL((gqa_batch_kernel<F16, DK, DV, NWQ, NWK, TK, NS, OCC, EXTRA>), dim3((unsigned) (grid > p.n_wg ? grid : p.n_wg)), dim3(64 * NWQ * NWK), lds, st, p);
    if ((e = hipGetLastError()) != hipSuccess || p.own_lens || p.deal == WHOLE) return e;
    hipLaunchKernelGGL((gqa_batch_join_kernel<F16, DV, NWQ>), dim3((unsigned) p.n_wg, DV / 32), dim3(256), 0, st, p);
    return hipGetLastError();
}
// Heads of 192: tiles of 32 keys in three stages, so that two workgroups' lie in a CU's LDS; of 256: tiles of 32, so that a wave's scores leave room in its registers (6 x 700
// tokens, window and cap: 277 us with 64 keys, 235 with 32), in four stages (228 with two, 219 with four).  Narrower heads have two stages of 64: a third one for heads of 64 made
// 8 x 512 tokens behind 16384 rows 293 us, not 283.
template <bool F16, int DK, int DV, Extra EXTRA>
hipError_t launch_shape(const BatchP & p, const BatchPlan & pl, hipStream_t st) {
    if constexpr (DK <= 128) if (pl.shape == FOUR_KEYS) return launch_batch<F16, DK, DV, 1, 4, 128, 2, batch_wg_per_cu(DK, FOUR_KEYS, EXTRA == NOTHING), EXTRA>(p, pl, st);
    if (pl.shape == FOUR_ROWS) return launch_batch<F16, DK, DV, 4, 1, DK >= 192 ? 32 : 64, DK == 256 ? 4 : DK == 192 ? 3 : 2, batch_wg_per_cu(DK, FOUR_ROWS, EXTRA == NOTHING), EXTRA>(p, pl, st);
    return launch_batch<F16, DK, DV, 2, 2, 64, DK == 192 ? 3 : 2, batch_wg_per_cu(DK, TWO_TWO, EXTRA == NOTHING), EXTRA>(p, pl, st);
}
template <bool F16, Extra EXTRA>
hipError_t launch_widths(const BatchP & p, const BatchPlan & pl, int dk, hipStream_t st) {
    switch (dk) {
        case 64:  return launch_shape<F16, 64, 64, EXTRA>(p, pl, st);
        case 128: return launch_shape<F16, 128, 128, EXTRA>(p, pl, st);
        case 192: return launch_shape<F16, 192, 128, EXTRA>(p, pl, st);
        default:  return launch_shape<F16, 256, 256, EXTRA>(p, pl, st);
    }
}

}  // namespace

template <bool F16> hipError_t batch_launch(const BatchP & p, const BatchPlan & pl, int dk, hipStream_t st) {
    // (the mask in units of the products needs a scale that it can be divided by)
    if (p.cap_out != 0.f || (p.mask && !(p.scale_log2 > 1e-30f))) return launch_widths<F16, CAP>(p, pl, dk, st);
    return p.mask ? launch_widths<F16, MASK>(p, pl, dk, st) : launch_widths<F16, NOTHING>(p, pl, dk, st);
}

}  // namespace gqa
}  // namespace mla
