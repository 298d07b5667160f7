/* Expert routing (le_moe_route, le_moe_sort, le_moe_permute, le_moe_combine and their gradients, include/le_qmm.h). */
#include <hip/hip_runtime.h>

#include "le_f32_types.h"
#include "le_route_args.h"

static __device__ __forceinline__ float wave_sum(float v) {
    for (int o = 32; o > 0; o >>= 1) v += __shfl_xor(v, o);
    return v;
}

/* Top-k by one wave per token: lane l holds experts l, l + 64, ...; k rounds of a wave-wide maximum, the lowest expert of equal
 * ones first. Lane s < k keeps selection s. */
template <int TY> __device__ __forceinline__ void route_body(const RouteArgs &a, int t) {
    const int lane = threadIdx.x & 63;
    const typename XT<TY>::raw *l = (const typename XT<TY>::raw *)a.logits + (size_t)t * a.n_exp;
    float v[16];
#pragma unroll
    for (int j = 0; j < 16; j++) {
        const int e = 64 * j + lane;
        const float x = e < a.n_exp ? XT<TY>::up(l[e]) : -INFINITY;
        v[j] = x == x ? x : -INFINITY;
    }
    int my_e = -1;
    float my_v = -INFINITY;
    for (int r = 0; r < a.k; r++) {
        float mx = v[0];
#pragma unroll
        for (int j = 1; j < 16; j++) mx = fmaxf(mx, v[j]);
        for (int o = 32; o > 0; o >>= 1) mx = fmaxf(mx, __shfl_xor(mx, o));
        if (!(mx > -INFINITY)) break; /* uniform */
        int e = -1;
#pragma unroll
        for (int j = 0; j < 16; j++) {
            const unsigned long long b = __ballot(v[j] == mx);
            if (e < 0 && b) {
                const int wl = __ffsll((long long)b) - 1;
                e = 64 * j + wl;
                v[j] = lane == wl ? -INFINITY : v[j];
            }
        }
        if (lane == r) my_e = e, my_v = mx;
    }
    const float top = __shfl(my_v, 0);
    const float ex = lane < a.k && my_e >= 0 ? expf(my_v - top) : 0.f;
    const float tot = wave_sum(ex);
    if (lane < a.k) {
        a.idx[(size_t)t * a.k + lane] = my_e;
        a.w[(size_t)t * a.k + lane] = my_e >= 0 ? ex / tot : 0.f;
    }
}

template <int TY> __device__ __forceinline__ void route_bwd_body(const RouteBwdArgs &a, int t) {
    const int lane = threadIdx.x & 63;
    int e = -1;
    float w = 0.f, dw = 0.f;
    if (lane < a.k) {
        e = a.idx[(size_t)t * a.k + lane];
        if (e < 0 || e >= a.n_exp) e = -1;
        if (e >= 0) w = a.w[(size_t)t * a.k + lane], dw = a.dw[(size_t)t * a.k + lane];
    }
    const float g = w * (dw - wave_sum(w * dw));
    typename XT<TY>::raw *d = (typename XT<TY>::raw *)a.dlogits + (size_t)t * a.n_exp;
    for (int e0 = 0; e0 < a.n_exp; e0 += 64) {
        float v = 0.f;
        for (int s = 0; s < a.k; s++) {
            const int es = __shfl(e, s);
            const float gs = __shfl(g, s);
            if (es == e0 + lane) v += gs;
        }
        if (e0 + lane < a.n_exp) d[e0 + lane] = XT<TY>::down(v);
    }
}

/* One block per expert: the pairs of lower experts counted, then its own placed in pair order (ranks by ballots). The
 * block after the last expert marks the dropped pairs and writes off[n_exp]. */
extern "C" __global__ void __launch_bounds__(256) le_rt_sort(SortArgs a) {
    __shared__ int wcnt[4];
    const int e = blockIdx.x, lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    int low = 0;
    for (long long pl = threadIdx.x; pl < a.np; pl += 256) {
        const int p = (int)pl;
        const int v = a.idx[p];
        low += v >= 0 && v < e;
        if (e == a.n_exp && a.pos && (v < 0 || v >= e)) a.pos[p] = -1;
    }
    for (int o = 32; o > 0; o >>= 1) low += __shfl_xor(low, o);
    if (lane == 0) wcnt[wave] = low;
    __syncthreads();
    int at = wcnt[0] + wcnt[1] + wcnt[2] + wcnt[3];
    if (threadIdx.x == 0) a.off[e] = at;
    if (e == a.n_exp) return;
    for (long long p0 = 0; p0 < a.np; p0 += 256) {
        const bool in = p0 + threadIdx.x < a.np;
        const int p = in ? (int)(p0 + threadIdx.x) : 0;
        const bool hit = in && a.idx[p] == e;
        const unsigned long long b = __ballot(hit);
        __syncthreads();
        if (lane == 0) wcnt[wave] = __popcll(b);
        __syncthreads();
        int q = at + __popcll(b & ((1ull << lane) - 1ull));
        for (int w = 0; w < 4; w++) {
            q += w < wave ? wcnt[w] : 0;
            at += wcnt[w];
        }
        if (hit) {
            if (a.in_idx) a.in_idx[q] = p / a.k;
            if (a.out_idx) a.out_idx[q] = p;
            if (a.pos) a.pos[p] = q;
        }
    }
}

/* The expert row of pair p, or -1. */
static __device__ __forceinline__ int row_of(const RowsArgs &a, int p) {
    const int r = a.pos ? a.pos[p] : p;
    return r >= 0 && r < a.n_row ? r : -1;
}

/* One block per token. */
template <int TY> __device__ __forceinline__ void permute_body(const RowsArgs &a, int t) {
    const typename XT<TY>::raw *x = (const typename XT<TY>::raw *)a.src + (size_t)t * a.ldt;
    for (int s = 0; s < a.k; s++) {
        const int r = row_of(a, t * a.k + s);
        if (r < 0) continue;
        typename XT<TY>::raw *e = (typename XT<TY>::raw *)a.dst + (size_t)r * a.lde;
        for (int c = threadIdx.x; c < a.cols; c += 256) e[c] = x[c];
    }
}

template <int TY> __device__ __forceinline__ void combine_body(const RowsArgs &a, int t) {
    typename XT<TY>::raw *out = (typename XT<TY>::raw *)a.dst + (size_t)t * a.ldt;
    for (int c = threadIdx.x; c < a.cols; c += 256) {
        float sum = 0.f;
        for (int s = 0; s < a.k; s++) {
            const int r = row_of(a, t * a.k + s);
            if (r < 0) continue;
            const float v = XT<TY>::up(((const typename XT<TY>::raw *)a.src)[(size_t)r * a.lde + c]);
            sum += a.w ? a.w[t * a.k + s] * v : v;
        }
        out[c] = XT<TY>::down(sum);
    }
}

template <int TY> __device__ __forceinline__ void combine_bwd_body(const RowsArgs &a, int t) {
    __shared__ float part[4];
    const typename XT<TY>::raw *dout = (const typename XT<TY>::raw *)a.src + (size_t)t * a.ldt;
    for (int s = 0; s < a.k; s++) {
        const int p = t * a.k + s, r = row_of(a, p);
        if (r < 0) {
            if (a.dw && threadIdx.x == 0) a.dw[p] = 0.f;
            continue;
        }
        const float w = a.w ? a.w[p] : 1.f;
        const typename XT<TY>::raw *e = (const typename XT<TY>::raw *)a.e + (size_t)r * a.lde;
        typename XT<TY>::raw *de = (typename XT<TY>::raw *)a.dst + (size_t)r * a.lde;
        float dot = 0.f;
        for (int c = threadIdx.x; c < a.cols; c += 256) {
            const float d = XT<TY>::up(dout[c]);
            if (a.dw) dot += d * XT<TY>::up(e[c]);
            if (a.dst) de[c] = XT<TY>::down(w * d);
        }
        if (!a.dw) continue;
        dot = wave_sum(dot);
        __syncthreads();
        if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = dot;
        __syncthreads();
        if (threadIdx.x == 0) a.dw[p] = part[0] + part[1] + part[2] + part[3];
    }
}

/* Tokens of a wave (four waves a block) and of a block; the grid may be smaller than the tokens. */
#define WAVE_TOKENS for (long long t = blockIdx.x * 4ll + (threadIdx.x >> 6); t < a.n_tok; t += gridDim.x * 4ll)
#define BLOCK_TOKENS for (long long t = blockIdx.x; t < a.n_tok; t += gridDim.x)
#define LE_RT(TY)                                                                                                                      \
    extern "C" __global__ void __launch_bounds__(256) le_rt_route_##TY(RouteArgs a) { WAVE_TOKENS route_body<TY>(a, (int)t); }             \
    extern "C" __global__ void __launch_bounds__(256) le_rt_route_bwd_##TY(RouteBwdArgs a) { WAVE_TOKENS route_bwd_body<TY>(a, (int)t); }  \
    extern "C" __global__ void __launch_bounds__(256) le_rt_permute_##TY(RowsArgs a) { BLOCK_TOKENS permute_body<TY>(a, (int)t); }         \
    extern "C" __global__ void __launch_bounds__(256) le_rt_combine_##TY(RowsArgs a) { BLOCK_TOKENS combine_body<TY>(a, (int)t); }         \
    extern "C" __global__ void __launch_bounds__(256) le_rt_combine_bwd_##TY(RowsArgs a) { BLOCK_TOKENS combine_bwd_body<TY>(a, (int)t); }
LE_RT(0) LE_RT(1) LE_RT(30)
