// Values moved and joined within a wave's vector registers.
#pragma once

#include "thip_kernels_common.h"

namespace thip {

// A value moved within a wave's vector registers (what ds_bpermute does takes a trip to LDS, which counts where a workgroup's whole call is a few us);
// 0 where there is none to come.
template <int CONTROL, int ROWS = 0xf>
__device__ __forceinline__ int moved(int v) { return __builtin_amdgcn_update_dpp(0, v, CONTROL, ROWS, 0xf, true); }
template <int CONTROL, int ROWS = 0xf>
__device__ __forceinline__ float moved(float v) { return __uint_as_float((uint32_t)moved<CONTROL, ROWS>((int)__float_as_uint(v))); }

// Of 2 or 16 lanes next to one another, the same in each.
template <int LANES, typename F>
__device__ __forceinline__ float overLanes(float v, F &&f) {
    static_assert(LANES == 2 || LANES == 16);
    v = f(v, moved<0xb1>(v));  // the neighbour
    if constexpr (LANES == 16) {
        v = f(v, moved<0x4e>(v));   // the other pair of four
        v = f(v, moved<0x141>(v));  // the other four of eight, backwards
        v = f(v, moved<0x140>(v));  // the other eight of 16, backwards
    }
    return v;
}

__device__ __forceinline__ float maxOverHalves(float v) {
    const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
}
__device__ __forceinline__ float sumOverHalves(float v) {
    const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return __uint_as_float(r[0]) + __uint_as_float(r[1]);
}
// The pairs of rows of 16 lanes; of all four with the halves.
__device__ __forceinline__ float maxOverSixteens(float v) {
    const auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
}
__device__ __forceinline__ float sumOverSixteens(float v) {
    const auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return __uint_as_float(r[0]) + __uint_as_float(r[1]);
}
__device__ __forceinline__ float maxOverQuarters(float v) { return maxOverHalves(maxOverSixteens(v)); }
__device__ __forceinline__ float sumOverQuarters(float v) { return sumOverHalves(sumOverSixteens(v)); }

__device__ __forceinline__ int packBf16(float lo, float hi) { return __builtin_bit_cast(int, __builtin_convertvector((v2f){lo, hi}, v2bf)); }

}  // namespace thip
