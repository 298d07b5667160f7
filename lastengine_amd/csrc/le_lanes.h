/* Sums and maxima over groups of lanes without LDS (device). */
#pragma once

#include <hip/hip_runtime.h>

/* The value of the lane D away (1, 2), or of the mirrored lane of the 8 (4) or 16 (8) where all lanes of a 4 or 8 hold the same value by
 * then, or of the row 16 away: the steps of a butterfly over up to 32 lanes. */
template <int D> static __device__ __forceinline__ int lane_across(int v) {
    if constexpr (D == 1) return __builtin_amdgcn_mov_dpp(v, 0xB1, 0xf, 0xf, true);
    else if constexpr (D == 2) return __builtin_amdgcn_mov_dpp(v, 0x4E, 0xf, 0xf, true);
    else if constexpr (D == 4) return __builtin_amdgcn_mov_dpp(v, 0x141, 0xf, 0xf, true);
    else if constexpr (D == 8) return __builtin_amdgcn_mov_dpp(v, 0x140, 0xf, 0xf, true);
    else {
        const auto r = __builtin_amdgcn_permlane16_swap(v, v, false, false);
        return threadIdx.x & 16 ? r[0] : r[1];
    }
}
/* Over groups of N lanes, in every lane of them. */
template <int N, int D = 1> static __device__ __forceinline__ float lanes_sum(float v) {
    if constexpr (D < N) return lanes_sum<N, 2 * D>(v + __builtin_bit_cast(float, lane_across<D>(__builtin_bit_cast(int, v))));
    else return v;
}
template <int N, int D = 1> static __device__ __forceinline__ int lanes_sum(int v) {
    if constexpr (D < N) return lanes_sum<N, 2 * D>(v + lane_across<D>(v));
    else return v;
}
template <int N, int D = 1> static __device__ __forceinline__ unsigned lanes_max(unsigned v) {
    if constexpr (D < N) return lanes_max<N, 2 * D>(max(v, (unsigned)lane_across<D>((int)v)));
    else return v;
}
