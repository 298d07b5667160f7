/* Matrix-vector products with 4-bit codes and group scales (le_matvec_g4, include/le_qmm.h):
 *     y[r] = sum over groups g of scale[r][g] * sum over the group's c of (code[r][c] - zero[r][g]) * a[c].
 *
 * le_g4_x*_s*_*: one wave per four rows, slot and token. Lane l takes 8 codes (one dword) of each 512, so a wave reads 256
 * contiguous bytes a step; products and sums in fp32. */
#include <hip/hip_runtime.h>

#include "le_f32_types.h"
#include "le_g4_args.h"

template <int XTY, int STY, bool SWIGLU> __device__ __forceinline__ void g4_row(const G4Args &a, int r) {
    const int lane = threadIdx.x & 63, s = blockIdx.y, t = blockIdx.z;
    if (r >= a.rows) return; /* uniform over the wave */
    const int mat = a.sel ? a.sel[s] : s;
    typename XT<XTY>::raw *y = (typename XT<XTY>::raw *)a.y + ((size_t)s * a.m + t) * a.rows + r;
    if (mat < 0 || mat >= a.n_mat) {
        if (lane == 0) *y = XT<XTY>::down(0.f);
        return;
    }
    const size_t row = (size_t)mat * a.rows + r;
    const unsigned *w = (const unsigned *)(a.codes + row * (a.cols / 2));
    const typename XT<STY>::raw *sc = (const typename XT<STY>::raw *)a.scales + row * a.ng;
    const typename XT<STY>::raw *zp = (const typename XT<STY>::raw *)a.zeros + row * a.ng;
    const typename XT<XTY>::raw *x = (const typename XT<XTY>::raw *)a.x + ((size_t)(s / a.share) * a.m + t) * a.xstride;
    float sum = 0.f;
    for (int d = lane; d < a.cols / 8; d += 64) {
        const int g = d * 8 / a.group;
        const float scale = XT<STY>::up(sc[g]), zero = a.zeros ? XT<STY>::up(zp[g]) : 8.f;
        const unsigned q = w[d];
        float part = 0.f;
#pragma unroll
        for (int i = 0; i < 8; i++) {
            const int c = d * 8 + i;
            float v = XT<XTY>::up(x[c]);
            if (SWIGLU) v = v / (1.f + expf(-v)) * XT<XTY>::up(x[a.cols + c]);
            part += ((float)((q >> 4 * i) & 15u) - zero) * v;
        }
        sum += scale * part;
    }
    for (int o = 32; o > 0; o >>= 1) sum += __shfl_xor(sum, o);
    if (lane == 0) *y = XT<XTY>::down(sum);
}

template <int XTY, int STY, bool SWIGLU> __device__ __forceinline__ void g4_body(const G4Args &a) {
    for (int i = 0; i < 4; i++) g4_row<XTY, STY, SWIGLU>(a, (blockIdx.x * 4 + (threadIdx.x >> 6)) * 4 + i);
}

#define LE_G4(X, S)                                                                                              \
    extern "C" __global__ void __launch_bounds__(256) le_g4_x##X##_s##S##_plain(G4Args a) { g4_body<X, S, false>(a); } \
    extern "C" __global__ void __launch_bounds__(256) le_g4_x##X##_s##S##_swiglu(G4Args a) { g4_body<X, S, true>(a); }
LE_G4(0, 0) LE_G4(0, 1) LE_G4(0, 30) LE_G4(1, 0) LE_G4(1, 1) LE_G4(1, 30) LE_G4(30, 0) LE_G4(30, 1) LE_G4(30, 30)
