/* Low-rank adapters beside a shared projection (le_lora, include/le_qmm.h), compiled once per type of the activations (LE_LO_XTY).
 * Two launches: u[t] = scale A x[t] over the columns, then y[t] = base[t] + B u[t] over the rank. */
#include <hip/hip_runtime.h>

#include "le_f32_types.h"
#include "le_lora_args.h"

#define LE_GLOBAL __attribute__((address_space(1)))

namespace {

constexpr int XTY = LE_LO_XTY;
using X = XT<XTY>::raw;

__device__ __forceinline__ float ld_x(const void *p, long long i) { return XT<XTY>::up(((const LE_GLOBAL X *)p)[i]); }
template <int WTY> __device__ __forceinline__ float ld_w(const void *p, long long i) {
    return XT<WTY>::up(((const LE_GLOBAL typename XT<WTY>::raw *)p)[i]);
}
/* The adapter of token t, -1: none. */
__device__ __forceinline__ int adapter(const LoraArgs &a, int t) {
    const int i = ((const LE_GLOBAL int *)a.idx)[t];
    return i >= 0 && i < a.n_ad ? i : -1;
}

template <int WTY> __device__ __forceinline__ void down_body(const LoraArgs &a) {
    const int l = threadIdx.x & 63;
    for (long long p = blockIdx.x * 4LL + (threadIdx.x >> 6); p < (long long)a.m * a.rank; p += gridDim.x * 4LL) {
        const int t = (int)(p / a.rank), j = (int)(p % a.rank), ad = adapter(a, t);
        if (ad < 0) continue;
        float s = 0.f;
        for (int c = l; c < a.cols; c += 64) s += ld_w<WTY>(a.a, ((long long)ad * a.rank + j) * a.cols + c) * ld_x(a.x, t * a.ldx + c);
#pragma unroll
        for (int d = 32; d; d >>= 1) s += __shfl_xor(s, d);
        if (l == 0) ((LE_GLOBAL float *)a.u)[p] = s * (a.scale ? ((const LE_GLOBAL float *)a.scale)[ad] : 1.f);
    }
}
template <int WTY> __device__ __forceinline__ void up_body(const LoraArgs &a) {
    const int r = blockIdx.x * 256 + threadIdx.x;
    if (r >= a.rows) return;
    for (int t = blockIdx.y; t < a.m; t += gridDim.y) {
        const int ad = adapter(a, t);
        float s = 0.f;
        if (ad >= 0)
            for (int j = 0; j < a.rank; j++) s += ld_w<WTY>(a.b, ((long long)ad * a.rows + r) * a.rank + j) * ((const LE_GLOBAL float *)a.u)[(long long)t * a.rank + j];
        ((LE_GLOBAL X *)a.y)[t * a.ldy + r] = XT<XTY>::down(a.base ? ld_x(a.base, t * a.ldb + r) + s : s);
    }
}

}  // namespace

#define LE_LO_NAME2(WHAT, X, W) le_lo_##WHAT##_##X##_##W
#define LE_LO_NAME(WHAT, X, W) LE_LO_NAME2(WHAT, X, W)
#define LE_LO(W)                                                                                                              \
    extern "C" __global__ void __launch_bounds__(256) LE_LO_NAME(down, LE_LO_XTY, W)(LoraArgs a) { down_body<W>(a); } \
    extern "C" __global__ void __launch_bounds__(256) LE_LO_NAME(up, LE_LO_XTY, W)(LoraArgs a) { up_body<W>(a); }
LE_LO(0)
LE_LO(1)
LE_LO(30)
