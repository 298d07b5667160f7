/* Residual, RMS norm and int8 activations in one launch (le_add_rms_quant, include/le_qmm.h).
 *
 * A row is read once and stays in registers from the sum of its squares to its codes: L lanes a row (a wave, or a block of 256 or 1024),
 * NC pieces of 16 bytes a lane, a unit of 32 values in 8 (16-bit types: 4) lanes. Bound by memory for many rows. The sum, the root and the first
 * product are in 64 bits, which the memory's time covers: the codes are then those of the formula whatever L is, and the largest
 * fp32 values need no scaling. 16-bit rows are held as fp32, for which four pieces in each of 1024 lanes (rows of 16385 to 32768 values) have 11
 * registers too few (48 bytes of scratch a lane). Rows of more than four pieces in each of 1024
 * lanes, and rows that end inside a piece (no codes then), are read twice. */
#include <hip/hip_runtime.h>

#include "le_f32_types.h"
#include "le_lanes.h"
#include "le_norm_args.h"

#define LE_GLOBAL __attribute__((address_space(1)))

namespace {

typedef unsigned v4u __attribute__((ext_vector_type(4)));
/* 16 bytes at any address of values of S bytes */
template <int S> struct Any;
template <> struct Any<2> { typedef v4u __attribute__((aligned(2))) v; };
template <> struct Any<4> { typedef v4u __attribute__((aligned(4))) v; };

/* A piece's values: all, or the n that there are (zeros behind them); TAIL: n may also lie between.
 * ONCE: read by nobody else after this (not kept in the caches: 4096 x 4096, x, res and o of fp32 82 -> 63 us, of bf16 48 -> 38; but a row's first
 * reading of two keeps it: x, res, h and o of 4096 x 4097 fp32 90 -> 76 us, of 8192 x 1001 bf16 35 -> 28, 64 x 40000 fp32 with codes 28 -> 22). */
template <int TY, int V, bool TAIL, bool ONCE> __device__ __forceinline__ void load(const void *p, long long at, int n, float *v) {
    using T = typename XT<TY>::raw;
    const LE_GLOBAL T *g = (const LE_GLOBAL T *)p + at;
    if (n >= V) {
        typedef const LE_GLOBAL typename Any<sizeof(T)>::v *from;
        const v4u w = ONCE ? __builtin_nontemporal_load((from)g) : *(from)g;
#pragma unroll
        for (int i = 0; i < V; i++) {
            const unsigned word = w[V == 4 ? i : i >> 1];
            if constexpr (V == 4) v[i] = __builtin_bit_cast(float, word);
            else v[i] = XT<TY>::up((T)(word >> (i & 1) * 16));
        }
    } else {
#pragma unroll
        for (int i = 0; i < V; i++) v[i] = TAIL && i < n ? XT<TY>::up(g[i]) : 0.f;
    }
}
template <int TY, int V, bool TAIL> __device__ __forceinline__ void store(void *p, long long at, int n, const float *v) {
    using T = typename XT<TY>::raw;
    LE_GLOBAL T *g = (LE_GLOBAL T *)p + at;
    if (n >= V) {
        v4u w;
#pragma unroll
        for (int d = 0; d < 4; d++) {
            if constexpr (V == 4) w[d] = __builtin_bit_cast(unsigned, v[d]);
            else w[d] = XT<TY>::down(v[2 * d]) | (unsigned)XT<TY>::down(v[2 * d + 1]) << 16;
        }
        *(LE_GLOBAL typename Any<sizeof(T)>::v *)g = w;
    } else if constexpr (TAIL) {
#pragma unroll
        for (int i = 0; i < V; i++)
            if (i < n) g[i] = XT<TY>::down(v[i]);
    }
}

/* h from here on, as it is stored. ONCE: of load() */
template <int TY, int V, bool TAIL, bool ONCE> __device__ __forceinline__ void sum_with(const NormArgs &a, long long t, int i, float *v) {
    load<TY, V, TAIL, ONCE>(a.x, t * a.ldx + i, a.n - i, v);
    if (a.res) {
        float r[V];
        load<TY, V, TAIL, ONCE>(a.res, t * a.ldr + i, a.n - i, r);
#pragma unroll
        for (int j = 0; j < V; j++) v[j] = XT<TY>::up(XT<TY>::down(v[j] + r[j]));
    }
}

/* 1 / sqrt of the mean, NaN where it is not finite */
__device__ __forceinline__ double root(const NormArgs &a, double s) {
    const double mean = s / a.n + a.eps;
    return s < __builtin_inf() && mean > 0.0 ? 1.0 / sqrt(mean) : __builtin_nan("");
}

/* The norm of a piece, and its codes */
template <int TY, int V, bool TAIL> __device__ __forceinline__ void finish(const NormArgs &a, long long t, int i, const float *h, double r) {
    constexpr int UNIT = 32 / V; /* lanes of 32 values */
    float w[V], o[V];
    unsigned am = 0; /* the largest |o| as bits, whose order is that of the values, NaN behind infinity */
    load<0, 4, TAIL, false>(a.w, i, a.n - i, w);
    if constexpr (V == 8) load<0, 4, TAIL, false>(a.w, i + 4, a.n - i - 4, w + 4);
#pragma unroll
    for (int j = 0; j < V; j++) {
        o[j] = (float)((double)h[j] * r) * w[j];
        am = max(am, __builtin_bit_cast(unsigned, o[j]) & 0x7FFFFFFFu);
    }
    const int n = a.n - i;
    if (n > 0) {
        if (a.h) store<TY, V, TAIL>(a.h, t * a.ldh + i, n, h);
        if (a.o) store<TY, V, TAIL>(a.o, t * a.ldo + i, n, o);
    }
    if (a.xq) { /* n is a multiple of 32: whole units */
        am = lanes_max<UNIT>(am);
        const bool fine = am < 0x7F800000u;
        /* 1 / d is infinite for d below 2^-128: both sides of such units are taken 2^64 times as large, which changes no bit of the others' product */
        const float d = __builtin_bit_cast(float, am) / 127.0f, up = d < 0x1p-126f ? 0x1p64f : 1.0f, id = d > 0.f ? 1.0f / (d * up) : 0.f;
        int sum = 0;
        unsigned q[V / 4];
#pragma unroll
        for (int j = 0; j < V; j++) {
            const int c = (int)fminf(fmaxf(rintf(o[j] * up * id), -127.f), 127.f);
            sum += c;
            q[j >> 2] = j & 3 ? q[j >> 2] | (c & 255) << 8 * (j & 3) : c & 255;
        }
        sum = fine ? lanes_sum<UNIT>(sum) : 0;
#pragma unroll
        for (int j = 0; j < V / 4; j++) q[j] = fine ? q[j] : 0;
        if (n > 0) {
            typedef unsigned __attribute__((aligned(1))) word;
            typedef unsigned long long __attribute__((aligned(1))) words;
            LE_GLOBAL signed char *xq = (LE_GLOBAL signed char *)a.xq + t * a.n + i;
            if constexpr (V == 4) *(LE_GLOBAL word *)xq = q[0];
            else *(LE_GLOBAL words *)xq = q[0] | (unsigned long long)q[V / 4 - 1] << 32;
            if ((i & 31) == 0) {
                ((LE_GLOBAL float *)a.xd)[(t * a.n + i) >> 5] = d;
                if (a.xs) ((LE_GLOBAL int *)a.xs)[(t * a.n + i) >> 5] = sum;
            }
        }
    }
}

template <int L> __device__ __forceinline__ double row_sum(double s, double *part) {
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) s += __shfl_xor(s, d);
    if constexpr (L > 64) {
        __syncthreads();
        if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = s;
        __syncthreads();
        s = part[0];
#pragma unroll
        for (int w = 1; w < L / 64; w++) s += part[w];
    }
    return s;
}

template <int TY, int L, int NC> __device__ __forceinline__ void norm_body(const NormArgs &a) {
    constexpr int V = TY == 0 ? 4 : 8, ROWS = L == 64 ? 4 : 1; /* rows a block */
    __shared__ double part[L / 64];
    const int l = threadIdx.x & (L - 1);
    for (long long t = (long long)blockIdx.x * ROWS + threadIdx.x / L; t < a.m; t += (long long)gridDim.x * ROWS) {
        float h[NC][V];
        double s = 0.0;
#pragma unroll
        for (int c = 0; c < NC; c++) sum_with<TY, V, false, true>(a, t, (l + L * c) * V, h[c]);
#pragma unroll
        for (int c = 0; c < NC; c++)
#pragma unroll
            for (int j = 0; j < V; j++) s = fma((double)h[c][j], (double)h[c][j], s);
        const double r = root(a, row_sum<L>(s, part));
#pragma unroll
        for (int c = 0; c < NC; c++) finish<TY, V, false>(a, t, (l + L * c) * V, h[c], r);
    }
}
template <int TY, int L> __device__ __forceinline__ void any_body(const NormArgs &a) {
    constexpr int V = TY == 0 ? 4 : 8;
    __shared__ double part[L / 64];
    for (long long t = blockIdx.x; t < a.m; t += gridDim.x) {
        double s = 0.0;
        for (int i = threadIdx.x * V; i < a.n; i += L * V) {
            float h[V];
            sum_with<TY, V, true, false>(a, t, i, h);
#pragma unroll
            for (int j = 0; j < V; j++) s = fma((double)h[j], (double)h[j], s);
        }
        const double r = root(a, row_sum<L>(s, part));
        for (int i0 = 0; i0 < a.n; i0 += L * V) { /* all lanes go along: units lie across them */
            const int i = i0 + threadIdx.x * V;
            float h[V];
            sum_with<TY, V, true, true>(a, t, i, h);
            finish<TY, V, true>(a, t, i, h, r);
        }
    }
}

}  // namespace

#define LE_NQ(TY, L, NC) \
    extern "C" __global__ void __launch_bounds__(L == 64 ? 256 : L) le_nq_##TY##_l##L##_c##NC(NormArgs a) { norm_body<TY, L, NC>(a); }
#define LE_NQ_ALL(TY)                                                                                             \
    LE_NQ(TY, 64, 1) LE_NQ(TY, 64, 2) LE_NQ(TY, 256, 1) LE_NQ(TY, 256, 2) LE_NQ(TY, 256, 4)                        \
    LE_NQ(TY, 1024, 1) LE_NQ(TY, 1024, 2) LE_NQ(TY, 1024, 4)                                                      \
    extern "C" __global__ void __launch_bounds__(256) le_nq_##TY##_any256(NormArgs a) { any_body<TY, 256>(a); }   \
    extern "C" __global__ void __launch_bounds__(1024) le_nq_##TY##_any1024(NormArgs a) { any_body<TY, 1024>(a); }
LE_NQ_ALL(0)
LE_NQ_ALL(1)
LE_NQ_ALL(30)
