// What a layer does to its new queries, keys and values before attention over a paged cache of ordinary heads (include/gqa_attn.h), in one
// pass for gfx950: RMS norm of every head's row, rotation, and the cache write.
//
// HBM-bound: every value is read once and written once, about 8 flops each.  A lane holds 8 consecutive values of a head's row (16 or 32
// bytes a load), 8 to 32 lanes a row; the sum of squares and the partners of a NeoX pair (half the rotated width away) come from
// other lanes by shuffles, so a row never touches LDS.  The (cos, sin) table of a token is built once by its workgroup: the position times
// the frequency in turns, in 64 bits, of which only the fraction of a turn is kept -- a far position costs no accuracy -- and the
// sine and cosine of that in f32.  8111 tokens of 32 + 8 + 8 rows of 128 in bf16: 44 us = 4.5 TB/s (a large copy: 4.9).

#include <math.h>

#include "gqa_common.hpp"
#include "../../include/mla_front.h"

using namespace mla;
using namespace mla::gqa;

namespace {

constexpr int MAX_PAIRS = 128;
// Below this a token's sets of rows have workgroups of their own, from there on one workgroup takes them all and makes the table once.  A whole call,
// 40 rows of 128: 1 token 6.9 against 8.3 us, 256 tokens 6.4 against 7.6; 2048 tokens 17.2 against 17.4, 8192 tokens 50.8 against 44.3.
constexpr int FEW_TOKENS = 1024;

enum { T_F32 = 0, T_F16 = 1, T_BF16 = 2 };

struct Rows { const char * src; int64_t nb1, nb2; };

struct FrontP {
    Rows q, k, v;
    const char * qw, * kw;
    char * q_dst; int64_t qd_nb1, qd_nb2;
    char * kc; int64_t k_page, k_row, k_head;
    char * vc; int64_t v_page, v_row, v_head;
    int64_t n_pages, bt_stride;
    const int32_t * block_table, * seq_ids, * slots, * pos;
    const float * ff;
    int   n_tok, n_head, n_head_kv, dk, dv, n_dims, neox, n_seq;
    int   w_type, dst_type;
    float eps, inv_dk, mscale;
    double turns[MAX_PAIRS];      // frequency of a pair, turns per position (YaRN blended in)
};

template <int T> struct Raw8 { u32x4 a, b; };                     // 8 values as loaded (16-bit types: a alone)
template <int T> __device__ __forceinline__ Raw8<T> load8(const char * p) {
    Raw8<T> r;
    r.a = *(const u32x4 *) p;
    if constexpr (T == T_F32) r.b = *(const u32x4 *) (p + 16);
    return r;
}
template <int T> __device__ __forceinline__ void unpack8(const Raw8<T> & r, float (&x)[8]) {
#pragma unroll
    for (int i = 0; i < 8; i++) {
        if constexpr (T == T_F32)       x[i] = __uint_as_float(i < 4 ? r.a[i] : r.b[i - 4]);
        else if constexpr (T == T_F16)  x[i] = f16_bits_to_f32((r.a[i >> 1] >> (16 * (i & 1))) & 0xffffu);
        else                            x[i] = __uint_as_float((i & 1) ? r.a[i >> 1] & 0xffff0000u : r.a[i >> 1] << 16);
    }
}
__device__ __forceinline__ void load_weights(const char * w, int type, int at, float (&x)[8]) {
    if (type == T_F32)      { const Raw8<T_F32> r = load8<T_F32>(w + (int64_t) at * 4); unpack8<T_F32>(r, x); }
    else if (type == T_F16) { const Raw8<T_F16> r = load8<T_F16>(w + (int64_t) at * 2); unpack8<T_F16>(r, x); }
    else                    { const Raw8<T_BF16> r = load8<T_BF16>(w + (int64_t) at * 2); unpack8<T_BF16>(r, x); }
}
template <bool F16> __device__ __forceinline__ u32x4 pack8(const float (&x)[8]) {
    return u32x4{ pair16<F16>(x[0], x[1]), pair16<F16>(x[2], x[3]), pair16<F16>(x[4], x[5]), pair16<F16>(x[6], x[7]) };
}
__device__ __forceinline__ void store8(char * to, int type, const float (&x)[8]) {
    if (type == T_F16)       *(u32x4 *) to = pack8<true>(x);
    else if (type == T_BF16) *(u32x4 *) to = pack8<false>(x);
    else { *(f32x4 *) to = f32x4{ x[0], x[1], x[2], x[3] }; *(f32x4 *) (to + 16) = f32x4{ x[4], x[5], x[6], x[7] }; }
}

// Cache row of a token: page base and row of the page, or page -1
__device__ __forceinline__ int64_t page_of(const FrontP & p, int t, int & row) {
    const int slot = p.slots ? p.slots[t] : p.pos[t], seq = p.seq_ids[t];
    row = 0;
    if (slot < 0 || seq < 0 || seq >= p.n_seq || slot / MLA_PAGE_TOKENS >= p.bt_stride) return -1;
    const int64_t page = p.block_table[(int64_t) seq * p.bt_stride + slot / MLA_PAGE_TOKENS];
    row = slot % MLA_PAGE_TOKENS;
    return page < 0 || page >= p.n_pages ? -1 : page;
}

// Grid: (tokens, parts); LPR lanes a row of dk values (the power of two that holds dk / 8).  A workgroup takes every parts-th set of 256 / LPR rows
// of its token, SETS of them at a time whose loads are all under way while the table is made, and part 0 the values.
template <int SRC, bool KV_F16, int LPR, int SETS>
__global__ void __launch_bounds__(256) gqa_norm_rope_kernel(const FrontP p) {
    __shared__ float2 cs[MAX_PAIRS];
    constexpr int ROWS = 256 / LPR, ES = SRC == T_F32 ? 4 : 2;
    const int t = blockIdx.x, parts = gridDim.y;
    const int sub = threadIdx.x % LPR, r0 = threadIdx.x / LPR;
    const int e0 = sub * 8;
    const bool live = e0 < p.dk;
    const int  n_rows = p.n_head + (p.k.src ? p.n_head_kv : 0), n_sets = (n_rows + ROWS - 1) / ROWS;
    const int  half = p.n_dims / 2;
    Raw8<SRC> raw[SETS], val;
    auto load_sets = [&](int set0) {                               // (sets past the last repeat it)
#pragma unroll
        for (int i = 0; i < SETS; i++) {
            const int  r = min(min(set0 + i * parts, n_sets - 1) * ROWS + r0, n_rows - 1);
            const bool isq = r < p.n_head;
            const char * src = (isq ? p.q.src : p.k.src) + (int64_t) t * (isq ? p.q.nb2 : p.k.nb2) + (int64_t) (isq ? r : r - p.n_head) * (isq ? p.q.nb1 : p.k.nb1);
            if (i == 0 || set0 + i * parts < n_sets) raw[i] = load8<SRC>(src + (live ? e0 : 0) * ES);
        }
    };
    load_sets(blockIdx.y);
    // values: runs of 8, the first 256 of them ahead like the rows
    const int  per = p.dv / 8, n_val = p.v.src && blockIdx.y == 0 ? p.n_head_kv * per : 0;
    auto val_at = [&](int i) { const int h = i / per, c = i - h * per; return p.v.src + (int64_t) t * p.v.nb2 + (int64_t) h * p.v.nb1 + c * 8 * ES; };
    if ((int) threadIdx.x < n_val) val = load8<SRC>(val_at(threadIdx.x));
    float gq[8], gk[8];                                            // the weights of this lane's values
    if (p.qw) load_weights(p.qw, p.w_type, live ? e0 : 0, gq);
    if (p.kw) load_weights(p.kw, p.w_type, live ? e0 : 0, gk);
    const int pos = p.pos[t];
    int     row = 0;
    const int64_t page = p.k.src ? page_of(p, t, row) : -1;
    for (int i = threadIdx.x; i < half; i += 256) {
        double f = p.turns[i];
        if (p.ff) f /= (double) p.ff[i];
        const double a = (double) pos * f;
        const float  w = (float) (a - rint(a));                    // a fraction of a turn, in [-1/2, 1/2]
        cs[i] = make_float2(cospif(2.f * w) * p.mscale, sinpif(2.f * w) * p.mscale);
    }
    if (page >= 0)
        for (int i = threadIdx.x; i < n_val; i += 256) {           // as they are
            const int h = i / per, c = i - h * per;
            if (i >= 256) val = load8<SRC>(val_at(i));
            float x[8];
            unpack8<SRC>(val, x);
            *(u32x4 *) (p.vc + page * p.v_page + row * p.v_row + h * p.v_head + c * 16) = pack8<KV_F16>(x);
        }
    __syncthreads();
    for (int set0 = blockIdx.y; set0 < n_sets; set0 += SETS * parts) {
        if (set0 != (int) blockIdx.y) load_sets(set0);
#pragma unroll
        for (int i = 0; i < SETS; i++) {                           // (every lane of a wave takes part in the shuffles)
            if (set0 + i * parts >= n_sets) break;
            const int  r = (set0 + i * parts) * ROWS + r0;
            const bool has = r < n_rows, isq = r < p.n_head;
            float x[8];
            unpack8<SRC>(raw[i], x);
            if (isq ? p.qw != nullptr : p.kw != nullptr) {
                float ss = 0.f;
                if (live)
#pragma unroll
                    for (int e = 0; e < 8; e++) ss = fmaf(x[e], x[e], ss);
#pragma unroll
                for (int d = 1; d < LPR; d <<= 1) ss += __shfl_xor(ss, d, 64);
                const float ms = fmaf(ss, p.inv_dk, p.eps);                              // (the instruction takes numbers below 2^-126 for 0)
                const float inv = ms < 0x1p-100f ? __builtin_amdgcn_rsqf(ms * 0x1p64f) * 0x1p32f : __builtin_amdgcn_rsqf(ms);    // (off by 2^-23 of itself at most)
#pragma unroll
                for (int e = 0; e < 8; e++) x[e] = x[e] * inv * (isq ? gq[e] : gk[e]);
            }
            if (half) {
                float y[8];
                if (p.neox) {
                    // the other half of a pair: value e0 + n_dims/2 for the first half, e0 - n_dims/2 for the second (n_dims/2 a multiple of 8)
                    const bool low = e0 < half, in = e0 < p.n_dims;
                    const int  from = (int) (threadIdx.x & 63) + (in ? (low ? half / 8 : -(half / 8)) : 0);
#pragma unroll
                    for (int e = 0; e < 8; e++) y[e] = __shfl(x[e], from, 64);
                    if (in)
#pragma unroll
                        for (int e = 0; e < 8; e++) {
                            const float2 c = cs[low ? e0 + e : e0 - half + e];
                            x[e] = low ? fmaf(x[e], c.x, -y[e] * c.y) : fmaf(y[e], c.y, x[e] * c.x);
                        }
                } else if (e0 < p.n_dims) {
#pragma unroll
                    for (int e = 0; e < 8; e += 2) {
                        const float2 c = cs[(e0 + e) / 2];
                        const float  a = x[e], b = x[e + 1];
                        x[e] = fmaf(a, c.x, -b * c.y); x[e + 1] = fmaf(a, c.y, b * c.x);
                    }
                }
            }
            if (!has || !live) continue;
            if (isq) store8(p.q_dst + (int64_t) t * p.qd_nb2 + (int64_t) r * p.qd_nb1 + e0 * (p.dst_type == T_F32 ? 4 : 2), p.dst_type, x);
            else if (page >= 0) *(u32x4 *) (p.kc + page * p.k_page + row * p.k_row + (r - p.n_head) * p.k_head + e0 * 2) = pack8<KV_F16>(x);
        }
    }
}

int type_of(int ggml) { return ggml == MLA_TYPE_F32 ? T_F32 : ggml == MLA_TYPE_F16 ? T_F16 : T_BF16; }
bool known(int ggml) { return ggml == MLA_TYPE_F32 || ggml == MLA_TYPE_F16 || ggml == MLA_TYPE_BF16; }

template <int SRC, bool KV_F16, int LPR>
void launch_lanes(const FrontP & p, hipStream_t st) {
    const int rows = 256 / LPR, sets = (p.n_head + (p.k.src ? p.n_head_kv : 0) + rows - 1) / rows;
    if (p.n_tok < FEW_TOKENS) hipLaunchKernelGGL((gqa_norm_rope_kernel<SRC, KV_F16, LPR, 1>), dim3((unsigned) p.n_tok, (unsigned) (sets < 64 ? sets : 64)), dim3(256), 0, st, p);
    else                      hipLaunchKernelGGL((gqa_norm_rope_kernel<SRC, KV_F16, LPR, 4>), dim3((unsigned) p.n_tok), dim3(256), 0, st, p);
}
template <int SRC, bool KV_F16>
void launch_rows(const FrontP & p, hipStream_t st) {
    if (p.dk <= 64)       launch_lanes<SRC, KV_F16, 8>(p, st);
    else if (p.dk <= 128) launch_lanes<SRC, KV_F16, 16>(p, st);
    else                  launch_lanes<SRC, KV_F16, 32>(p, st);
}
template <bool KV_F16>
void launch_src(const FrontP & p, int src, hipStream_t st) {
    if (src == T_F32)      launch_rows<T_F32, KV_F16>(p, st);
    else if (src == T_F16) launch_rows<T_F16, KV_F16>(p, st);
    else                   launch_rows<T_BF16, KV_F16>(p, st);
}

int check_rows(const void * src, int64_t nb1, int64_t nb2) { return !al16(src) || (nb1 & 15) || (nb2 & 15) ? MLA_ERR_BAD_ALIGNMENT : 0; }
int check_pool(const gqa_pool & c) {
    if (!c.data) return MLA_ERR_NULL;
    if (!al16(c.data) || (c.nb_page & 15) || (c.nb_row & 15) || (c.nb_head & 15)) return MLA_ERR_BAD_ALIGNMENT;
    return c.nb_page < 0 || c.nb_row < 0 || c.nb_head < 0 ? MLA_ERR_BAD_SHAPE : 0;
}

}  // namespace

extern "C" int gqa_norm_rope_check(const gqa_norm_rope_args * a) {
    if (!a) return MLA_ERR_NULL;
    if (!known(a->src_type) || !known(a->w_type) || !known(a->dst_type)) return MLA_ERR_BAD_TYPE;
    if (a->k && a->kv_type != MLA_TYPE_F16 && a->kv_type != MLA_TYPE_BF16) return MLA_ERR_BAD_TYPE;
    if (a->n_tok < 0 || a->n_tok >= (1 << 24) || a->n_head < 1 || a->dk < 8 || a->dk % 8 || a->dk > 256) return MLA_ERR_BAD_SHAPE;
    if (a->k && (a->n_head_kv < 1 || a->n_seq < 0)) return MLA_ERR_BAD_SHAPE;
    if (a->v && (!a->k || a->dv < 8 || a->dv % 8 || a->dv > 256)) return MLA_ERR_BAD_SHAPE;
    if (a->mode != MLA_ROPE_MODE_NORM && a->mode != MLA_ROPE_MODE_NEOX) return MLA_ERR_UNSUPPORTED;
    if (a->n_dims < 0 || a->n_dims > a->dk || a->n_dims % (a->mode == MLA_ROPE_MODE_NEOX ? 16 : 8)) return MLA_ERR_BAD_SHAPE;
    if (a->n_dims && (!(a->freq_base > 1.0) || (a->ext_factor != 0.0 && (!(a->freq_scale > 0.0) || a->n_ctx_orig < 1 || !(a->beta_fast > 0.0) || !(a->beta_slow > 0.0)))))
        return MLA_ERR_UNSUPPORTED;
    if (a->n_tok == 0) return 0;
    if (!a->q || !a->q_dst || !a->pos) return MLA_ERR_NULL;
    int rc = check_rows(a->q, a->q_nb1, a->q_nb2);
    if (!rc) rc = check_rows(a->q_dst, a->qd_nb1, a->qd_nb2);
    if (!rc && a->q_weight) rc = check_rows(a->q_weight, 0, 0);
    if (rc) return rc;
    const int64_t apart = (const char *) a->q_dst - (const char *) a->q, row = (int64_t) a->dk * (a->src_type == MLA_TYPE_F32 ? 4 : 2), row_dst = (int64_t) a->dk * (a->dst_type == MLA_TYPE_F32 ? 4 : 2);
    if (apart == 0 ? a->src_type != a->dst_type || a->qd_nb1 != a->q_nb1 || a->qd_nb2 != a->q_nb2 : apart > -row_dst && apart < row) return MLA_ERR_UNSUPPORTED;
    if (a->k) {
        if (a->v && a->v_cache.data == a->k_cache.data) return a->v_cache.data ? MLA_ERR_UNSUPPORTED : MLA_ERR_NULL;
        if (!a->block_table || !a->seq_ids) return MLA_ERR_NULL;
        if (a->n_pages < 1 || a->bt_stride < 1) return MLA_ERR_BAD_SHAPE;
        if ((rc = check_rows(a->k, a->k_nb1, a->k_nb2)) || (rc = check_pool(a->k_cache))) return rc;
        if (a->k_weight && (rc = check_rows(a->k_weight, 0, 0))) return rc;
        if (a->v && ((rc = check_rows(a->v, a->v_nb1, a->v_nb2)) || (rc = check_pool(a->v_cache)))) return rc;
    }
    return 0;
}

extern "C" int gqa_norm_rope_launch(const gqa_norm_rope_args * a, void * stream) {
    const int rc = gqa_norm_rope_check(a);
    if (rc) return rc;
    if (a->n_tok == 0) return 0;
    FrontP p;
    p.q = Rows{ (const char *) a->q, a->q_nb1, a->q_nb2 };
    p.k = Rows{ (const char *) a->k, a->k_nb1, a->k_nb2 };
    p.v = Rows{ (const char *) a->v, a->v_nb1, a->v_nb2 };
    p.qw = (const char *) a->q_weight; p.kw = (const char *) a->k_weight;
    p.q_dst = (char *) a->q_dst; p.qd_nb1 = a->qd_nb1; p.qd_nb2 = a->qd_nb2;
    p.kc = (char *) a->k_cache.data; p.k_page = a->k_cache.nb_page; p.k_row = a->k_cache.nb_row; p.k_head = a->k_cache.nb_head;
    p.vc = (char *) a->v_cache.data; p.v_page = a->v_cache.nb_page; p.v_row = a->v_cache.nb_row; p.v_head = a->v_cache.nb_head;
    p.n_pages = a->n_pages; p.bt_stride = a->bt_stride; p.block_table = a->block_table; p.seq_ids = a->seq_ids; p.slots = a->slots; p.pos = a->pos;
    p.ff = a->freq_factors;
    p.n_tok = a->n_tok; p.n_head = a->n_head; p.n_head_kv = a->n_head_kv; p.dk = a->dk; p.dv = a->dv; p.n_dims = a->n_dims; p.n_seq = a->n_seq;
    p.neox = a->mode == MLA_ROPE_MODE_NEOX;
    p.w_type = type_of(a->w_type); p.dst_type = type_of(a->dst_type);
    p.eps = a->eps; p.inv_dk = 1.f / (float) a->dk; p.mscale = (float) a->attn_factor;
    // f_i = freq_base^(-2i / n_dims), scaled by freq_scale where YaRN interpolates (ggml/src/ggml-cpu/ggml-cpu.c:10272-10293, the
    // correction dims of ggml/src/ggml.c:3529-3541), in turns
    const double n = a->n_dims, base = a->freq_base, pi = 3.14159265358979323846;
    double lo = 0, hi = 0;
    if (a->n_dims && a->ext_factor != 0.0) {
        lo = fmax(0.0, floor(n * log(a->n_ctx_orig / (a->beta_fast * 2 * pi)) / (2 * log(base))));
        hi = fmin(n - 1, ceil(n * log(a->n_ctx_orig / (a->beta_slow * 2 * pi)) / (2 * log(base))));
        p.mscale = (float) (a->attn_factor * (1.0 + 0.1 * log(1.0 / a->freq_scale)));
    }
    // (a product per pair: 64 roundings in 64 bits are 1e-14 of the angle, 64 calls of pow are 3 us of every launch)
    const double ratio = a->n_dims ? pow(base, -2.0 / n) : 0.0;
    double f = 1.0 / (2 * pi);
    for (int i = 0; i < a->n_dims / 2; i++, f *= ratio) {
        double scale = a->freq_scale;
        if (a->ext_factor != 0.0) {
            const double mix = (1.0 - fmin(1.0, fmax(0.0, (i - lo) / fmax(0.001, hi - lo)))) * a->ext_factor;
            scale = scale * (1.0 - mix) + mix;
        }
        p.turns[i] = scale * f;
    }
    const int src = type_of(a->src_type);
    if (a->kv_type == MLA_TYPE_F16) launch_src<true>(p, src, (hipStream_t) stream);
    else                            launch_src<false>(p, src, (hipStream_t) stream);
    return (int) hipGetLastError();
}
