/* Residual, RMS norm and int8 activations in one launch (le_add_rms_quant, include/le_qmm.h). */
#include <hip/hip_runtime.h>

#include "le_f32_types.h"
#include "le_norm_args.h"

#define LE_GLOBAL __attribute__((address_space(1)))

namespace {

template <int TY> __device__ __forceinline__ float value(const void *p, long long i) {
    return XT<TY>::up(((const LE_GLOBAL typename XT<TY>::raw *)p)[i]);
}
/* x + res as it is stored */
template <int TY> __device__ __forceinline__ float sum_of(const NormArgs &a, long long t, int i) {
    const float x = value<TY>(a.x, t * a.ldx + i);
    return a.res ? XT<TY>::up(XT<TY>::down(x + value<TY>(a.res, t * a.ldr + i))) : x;
}

/* A block a row; a unit of 32 values by 32 lanes. */
template <int TY> __device__ __forceinline__ void norm_body(const NormArgs &a) {
    using T = typename XT<TY>::raw;
    __shared__ double part[4];
    for (long long t = blockIdx.x; t < a.m; t += gridDim.x) {
        double s = 0.0;
        for (int i = threadIdx.x; i < a.n; i += 256) {
            const double v = sum_of<TY>(a, t, i);
            s += v * v;
        }
#pragma unroll
        for (int d = 32; d; d >>= 1) s += __shfl_xor(s, d);
        __syncthreads();
        if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = s;
        __syncthreads();
        s = (part[0] + part[1]) + (part[2] + part[3]);
        const bool fine = s < __builtin_inf() && s / a.n + a.eps > 0.0;
        const double r = fine ? 1.0 / sqrt(s / a.n + a.eps) : __builtin_nan("");
        for (int i = threadIdx.x; i < (a.n + 31) / 32 * 32; i += 256) {
            const float h = i < a.n ? sum_of<TY>(a, t, i) : 0.f;
            const float o = i < a.n ? (float)((double)h * r) * ((const LE_GLOBAL float *)a.w)[i] : 0.f;
            if (i < a.n && a.h) ((LE_GLOBAL T *)a.h)[t * a.ldh + i] = XT<TY>::down(h);
            if (i < a.n && a.o) ((LE_GLOBAL T *)a.o)[t * a.ldo + i] = XT<TY>::down(o);
            if (a.xq) {
                float am = fabsf(o);
#pragma unroll
                for (int d = 16; d; d >>= 1) am = fmaxf(am, __shfl_xor(am, d, 32));
                const float dd = am / 127.0f, id = dd > 0.f ? 1.0f / dd : 0.f;
                const int q = fine ? (int)fminf(fmaxf(rintf(o * id), -127.f), 127.f) : 0;
                int sm = q;
#pragma unroll
                for (int d = 16; d; d >>= 1) sm += __shfl_xor(sm, d, 32);
                ((LE_GLOBAL signed char *)a.xq)[t * a.n + i] = (signed char)q;
                if ((i & 31) == 0) {
                    ((LE_GLOBAL float *)a.xd)[(t * a.n + i) / 32] = fine ? dd : __builtin_nanf("");
                    if (a.xs) ((LE_GLOBAL int *)a.xs)[(t * a.n + i) / 32] = sm;
                }
            }
        }
    }
}

}  // namespace

extern "C" __global__ void __launch_bounds__(256) le_nq_0(NormArgs a) { norm_body<0>(a); }
extern "C" __global__ void __launch_bounds__(256) le_nq_1(NormArgs a) { norm_body<1>(a); }
extern "C" __global__ void __launch_bounds__(256) le_nq_30(NormArgs a) { norm_body<30>(a); }
