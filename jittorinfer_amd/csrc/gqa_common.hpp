// Shared by the kernels of the paged cache of ordinary heads (include/gqa_attn.h; gfx950).
#pragma once

#include <atomic>

#include "mla_common.hpp"
#include "../../include/gqa_attn.h"

namespace mla {
namespace gqa {

constexpr int PAGE = MLA_PAGE_TOKENS;

// To 16 bits by the hardware's conversions, to nearest even (pack2's integer form of the bf16 rounding is six instructions a value).
template <bool F16> __device__ __forceinline__ unsigned short to16(float f) {
    if constexpr (F16) return bitcast<unsigned short>((_Float16) f);
    else               return bitcast<unsigned short>((__bf16) f);
}
template <bool F16> __device__ __forceinline__ unsigned pair16(float a, float b) { return to16<F16>(a) | ((unsigned) to16<F16>(b) << 16); }
template <bool F16> __device__ __forceinline__ float from16(unsigned short h) {
    if constexpr (F16) return (float) bitcast<_Float16>(h);
    else               return __uint_as_float((unsigned) h << 16);
}

// Sum over this lane and the ones before it.  Lanes take from their neighbours in the vector unit (shifts by 1, 2, 4, 8 inside a row of 16, then the
// last lane of a row to the next rows): eight instructions, where six shuffles through LDS are 600 cycles of latency.
__device__ __forceinline__ int scan_wave(int v) {
    v += __builtin_amdgcn_update_dpp(0, v, 0x111, 0xf, 0xf, false);
    v += __builtin_amdgcn_update_dpp(0, v, 0x112, 0xf, 0xf, false);
    v += __builtin_amdgcn_update_dpp(0, v, 0x114, 0xf, 0xf, false);
    v += __builtin_amdgcn_update_dpp(0, v, 0x118, 0xf, 0xf, false);
    v += __builtin_amdgcn_update_dpp(0, v, 0x142, 0xa, 0xf, false);
    v += __builtin_amdgcn_update_dpp(0, v, 0x143, 0xc, 0xf, false);
    return v;
}
// The value of lane `lane`, the same in every lane of the wave (`lane` too).
__device__ __forceinline__ int lane_of(int v, int lane) { return __builtin_amdgcn_readlane(v, lane); }

// What lanes of a wave have written to LDS is there for its other lanes, and what they have read may be overwritten.
__device__ __forceinline__ void wave_fence() {
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
}

// A score in log2 units from the product q . k, before the mask.  A soft cap c turns a score s into c tanh(y), y = s / c: 1 - 2 / (e^2y + 1) from y = 3/4 on,
// of which a small y would keep no digits; there s itself times tanh(y) / y, by Lambert's continued fraction to y^2 / 9 (off by y^10 / 10^7: 6e-9), so that a
// cap far above the scores leaves them as they are.  Either is off by 2^-21 of itself at most, and they share the reciprocal.
__device__ __forceinline__ float scaled_score(float scale_log2, float cap_in, float cap_out, float a) {
    const float s = scale_log2 * a;
    if (cap_out != 0.f) {
        const float y = fabsf(cap_in * a), u = y * y;
        const bool  small = y < 0.75f;
        const float r = __builtin_amdgcn_rcpf(small ? fmaf(u, fmaf(u, 15.f, 420.f), 945.f) : fast_exp2(2.f * LOG2E * y) + 1.f);
        return small ? s * (fmaf(u, u + 105.f, 945.f) * r) : copysignf(cap_out * fmaf(-2.f, r, 1.f), s);
    }
    return s;
}

// LDS over the 64 KB a kernel gets unasked: granted once a device, whatever it asks for later.
template <typename K> hipError_t grant_lds(K kernel, int lds, std::atomic<uint64_t> & granted) {
    if (lds < 60 * 1024) return hipSuccess;                       // (the kernels' own shared arrays come on top)
    int dev = 0;
    hipError_t e = hipGetDevice(&dev);
    if (e != hipSuccess) return e;
    const uint64_t bit = dev < 64 ? (uint64_t) 1 << dev : 0;
    if (!(granted.load(std::memory_order_relaxed) & bit)) {
        if ((e = hipFuncSetAttribute((const void *) kernel, hipFuncAttributeMaxDynamicSharedMemorySize, lds)) != hipSuccess) return e;
        granted.fetch_or(bit, std::memory_order_relaxed);
    }
    return hipSuccess;
}

inline bool al16(const void * ptr) { return ((uintptr_t) ptr & 15) == 0; }

}  // namespace gqa
}  // namespace mla
