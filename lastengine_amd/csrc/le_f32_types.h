/* Device loads and stores of the activation types (LE_F32 = 0, LE_F16 = 1, LE_BF16 = 30) as fp32. */
#pragma once

#include <hip/hip_runtime.h>

template <int TY> struct XT;
template <> struct XT<0> {
    using raw = float;
    static __device__ __forceinline__ float up(raw v) { return v; }
    static __device__ __forceinline__ raw down(float v) { return v; }
};
template <> struct XT<1> {
    using raw = unsigned short;
    static __device__ __forceinline__ float up(raw v) { return (float)__builtin_bit_cast(_Float16, v); }
    static __device__ __forceinline__ raw down(float v) { return __builtin_bit_cast(unsigned short, (_Float16)v); }
};
template <> struct XT<30> {
    using raw = unsigned short;
    static __device__ __forceinline__ float up(raw v) { return __builtin_bit_cast(float, (unsigned)v << 16); }
    /* round to nearest even (NaN stays NaN): the conversion instruction of gfx950 */
    static __device__ __forceinline__ raw down(float v) { return __builtin_bit_cast(unsigned short, (__bf16)v); }
};
