// Shared by the kernels of the paged cache of ordinary heads (include/gqa_attn.h; gfx950).
#pragma once

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

inline bool al16(const void * ptr) { return ((uintptr_t) ptr & 15) == 0; }

}  // namespace gqa
}  // namespace mla
