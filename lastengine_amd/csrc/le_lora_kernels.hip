/* Low-rank adapters beside a shared projection (le_lora, include/le_qmm.h), compiled once per type of the activations (LE_LO_XTY).
 * Two launches: u[t] = A x[t] over the columns, then y[t] = base[t] + B (scale u[t]) over the rank. Tokens are taken 16 at a time, as they
 * come; a tile of 16 with several adapters is done once for each of them, and what it gives for the others' tokens is dropped
 * (selected, so that nothing of one token or adapter reaches another). */
#include <hip/hip_runtime.h>

#include "le_f32_types.h"
#include "le_lora_args.h"

#define LE_GLOBAL __attribute__((address_space(1)))

namespace {

constexpr int XTY = LE_LO_XTY;
using X = XT<XTY>::raw;

typedef unsigned v4u __attribute__((ext_vector_type(4)));
typedef float v4f __attribute__((ext_vector_type(4)));
typedef _Float16 v8h __attribute__((ext_vector_type(8)));
typedef __bf16 v8b __attribute__((ext_vector_type(8)));

/* 16 bytes at any address of values of S bytes */
template <int S> struct Any;
template <> struct Any<2> { typedef v4u __attribute__((aligned(2))) v; };
template <> struct Any<4> { typedef v4u __attribute__((aligned(4))) v; };

/* ---- eight values of a row ---- */

template <int TY> struct Eight;
template <> struct Eight<0> {
    float v[8];
    __device__ __forceinline__ float up(int i) const { return v[i]; }
};
template <int TY> struct Eight {
    v4u v;
    __device__ __forceinline__ float up(int i) const { return XT<TY>::up((typename XT<TY>::raw)(v[i >> 1] >> (i & 1) * 16)); }
};
/* From p on, at any alignment of the type; zeros behind the n values that there are. */
template <int TY> __device__ __forceinline__ Eight<TY> load8(const void *base, long long at, int n) {
    using T = typename XT<TY>::raw;
    using v4u_any = typename Any<sizeof(T)>::v;
    const LE_GLOBAL T *p = (const LE_GLOBAL T *)base + at;
    Eight<TY> r;
    if constexpr (TY == 0) {
        if (n >= 8) {
            *(v4u *)&r.v[0] = *(const LE_GLOBAL v4u_any *)p;
            *(v4u *)&r.v[4] = *(const LE_GLOBAL v4u_any *)(p + 4);
        } else {
#pragma unroll
            for (int i = 0; i < 8; i++) r.v[i] = i < n ? p[i] : 0.f;
        }
    } else {
        if (n >= 8) {
            r.v = *(const LE_GLOBAL v4u_any *)p;
        } else {
            r.v = v4u{0, 0, 0, 0};
#pragma unroll
            for (int i = 0; i < 7; i++)
                if (i < n) r.v[i >> 1] |= (unsigned)p[i] << (i & 1) * 16;
        }
    }
    return r;
}

/* Value e of a 16-byte piece, and word d of the piece of values v. */
template <int TY> __device__ __forceinline__ float unpack(v4u v, int e) {
    const unsigned word = v[TY == 0 ? e : e >> 1];
    if constexpr (TY == 0) return __builtin_bit_cast(float, word);
    else return XT<TY>::up((typename XT<TY>::raw)(word >> (e & 1) * 16));
}
template <int TY> __device__ __forceinline__ unsigned pack(const float *v, int d) {
    if constexpr (TY == 0) return __builtin_bit_cast(unsigned, v[d]);
    else return XT<TY>::down(v[2 * d]) | (unsigned)XT<TY>::down(v[2 * d + 1]) << 16;
}

/* c += P Q^T over 32 of k: 16 rows of each, a lane's row l % 16 and its eight k from 8 (l / 16) on. Two operands of one 16-bit type
 * multiply as they are, others in fp32: either way the products are exact (fp32: a fused multiply-add's) and the sums fp32. */
template <int P, int Q> __device__ __forceinline__ v4f multiply(const Eight<P> &p, const Eight<Q> &q, v4f c) {
    if constexpr (P == 1 && Q == 1) {
        return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(v8h, p.v), __builtin_bit_cast(v8h, q.v), c, 0, 0, 0);
    } else if constexpr (P == 30 && Q == 30) {
        return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(v8b, p.v), __builtin_bit_cast(v8b, q.v), c, 0, 0, 0);
    } else {
#pragma unroll
        for (int i = 0; i < 8; i++) c = __builtin_amdgcn_mfma_f32_16x16x4f32(p.up(i), q.up(i), c, 0, 0, 0);
        return c;
    }
}

template <int N> struct Count { static constexpr int value = N; };

/* ---- the adapters of a tile ---- */

struct Tile {
    int t0;       /* first of its 16 tokens */
    int id;       /* adapter of this lane's token t0 + l % 16; -1: none, or no token */
    unsigned left; /* tokens whose adapter has not come yet */
    int cur;
    unsigned members; /* tokens of adapter cur */
    __device__ __forceinline__ Tile(const LoraArgs &a, int tile) {
        const int l = threadIdx.x & 63;
        t0 = tile * 16;
        const int t = t0 + (l & 15);
        id = t < a.m ? ((const LE_GLOBAL int *)a.idx)[t] : -1;
        if (id >= a.n_ad || id < 0) id = -1;
        left = (unsigned)__ballot(id >= 0) & 0xFFFF;
    }
    __device__ __forceinline__ bool next() {
        if (!left) return false;
        cur = __builtin_amdgcn_readlane(id, __ffs((int)left) - 1);
        members = (unsigned)__ballot(id == cur) & 0xFFFF;
        left &= ~members;
        return true;
    }
};

/* ---- down: u = A x ----
 * A block takes a tile, an adapter of it and a segment of the columns, its four waves 32 columns in turn; their sums meet in LDS. Rows of A
 * as the other operand, RF times 16 of them at once. Operands come straight from memory in the matrix instruction's layout, 64 (fp32:
 * 128) bytes in a row of each. */
template <int WTY, int RF> __device__ __forceinline__ void down_body(const LoraArgs &a) {
    __shared__ float part[4][RF][256];
    const int l = threadIdx.x & 63, wave = threadIdx.x >> 6, kl = (l >> 4) * 8;
    Tile t(a, blockIdx.x);
    const int s0 = blockIdx.z * a.steps, s1 = min(s0 + a.steps, (a.cols + 31) / 32), whole = min(s1, a.cols / 32);
    const long long xrow = min(t.t0 + (l & 15), a.m - 1) * a.ldx;
    for (int nth = 0; t.next(); nth++) {
        if (nth % gridDim.y != blockIdx.y) continue;
        for (int j0 = 0; j0 < a.rank; j0 += 16 * RF) {
            v4f c[RF];
            long long arow[RF];
#pragma unroll
            for (int f = 0; f < RF; f++) {
                c[f] = v4f{0.f, 0.f, 0.f, 0.f};
                arow[f] = ((long long)t.cur * a.rank + min(j0 + 16 * f + (l & 15), a.rank - 1)) * a.cols;
            }
            int s = s0 + wave;
            auto some = [&](auto count) { /* so many of the wave's steps, their loads ahead of their products */
                constexpr int U = decltype(count)::value;
                Eight<XTY> x[U];
                Eight<WTY> w[U][RF];
#pragma unroll
                for (int i = 0; i < U; i++) {
                    const int k = 32 * (s + 4 * i) + kl;
                    x[i] = load8<XTY>(a.x, xrow + k, 8);
#pragma unroll
                    for (int f = 0; f < RF; f++) w[i][f] = load8<WTY>(a.a, arow[f] + k, 8);
                }
#pragma unroll
                for (int i = 0; i < U; i++)
#pragma unroll
                    for (int f = 0; f < RF; f++) c[f] = multiply<XTY, WTY>(x[i], w[i][f], c[f]);
                s += 4 * U;
            };
            constexpr int U = RF == 4 ? 2 : 4;
            while (s + 4 * (U - 1) < whole) some(Count<U>());
            while (s < whole) some(Count<1>());
            if (s < s1) { /* the row's end */
                const int k = 32 * s + kl, n = a.cols - k;
                const Eight<XTY> x = load8<XTY>(a.x, xrow + k, n);
#pragma unroll
                for (int f = 0; f < RF; f++) c[f] = multiply<XTY, WTY>(x, load8<WTY>(a.a, arow[f] + k, n), c[f]);
            }
            __syncthreads();
#pragma unroll
            for (int f = 0; f < RF; f++)
#pragma unroll
                for (int i = 0; i < 4; i++) part[wave][f][((l >> 4) * 4 + i) * 16 + (l & 15)] = c[f][i];
            __syncthreads();
            const int row = threadIdx.x >> 4;
#pragma unroll
            for (int f = 0; f < RF; f++) {
                const int j = j0 + 16 * f + (threadIdx.x & 15);
                const float v = (part[0][f][threadIdx.x] + part[1][f][threadIdx.x]) + (part[2][f][threadIdx.x] + part[3][f][threadIdx.x]);
                if (j < a.rank && (t.members >> row & 1)) ((LE_GLOBAL float *)a.u)[((long long)blockIdx.z * a.m + t.t0 + row) * a.rank + j] = v;
            }
        }
    }
}

__device__ __forceinline__ float factor(const LoraArgs &a, int ad) { return a.scale ? ((const LE_GLOBAL float *)a.scale)[ad] : 1.f; }

/* ---- up, few tokens ----
 * A lane an output row, whose rank values of B it reads once for all tokens of the adapter; u in LDS. */
template <int WTY> __device__ __forceinline__ void upv_body(const LoraArgs &a) {
    extern __shared__ float lu[]; /* [token][rank, rounded up to 8] */
    const int rp = (a.rank + 7) & ~7, r = blockIdx.x * 256 + threadIdx.x, rc = min(r, a.rows - 1);
    Tile t(a, blockIdx.y);
    const LE_GLOBAL X *base = (const LE_GLOBAL X *)a.base;
    if (blockIdx.z == 0 && r < a.rows) { /* tokens of no adapter */
        for (unsigned none = ~t.left & 0xFFFF; none; none &= none - 1) {
            const int k = t.t0 + __ffs((int)none) - 1;
            if (k >= a.m) break;
            ((LE_GLOBAL X *)a.y)[k * a.ldy + r] = a.base ? base[k * a.ldb + r] : X(0);
        }
    }
    for (int nth = 0; t.next(); nth++) {
        if (nth % gridDim.z != blockIdx.z) continue;
        float b[16];
#pragma unroll
        for (int i = 0; i < 16; i++) b[i] = (t.members >> i & 1) && a.base ? XT<XTY>::up(base[(t.t0 + i) * a.ldb + rc]) : 0.f;
        const float f = factor(a, t.cur);
        __syncthreads();
        for (int id = threadIdx.x; id < 16 * rp; id += 256) {
            const int i = id / rp, j = id - i * rp;
            float v = 0.f;
            if ((t.members >> i & 1) && j < a.rank)
                for (int s = 0; s < a.segs; s++) v += ((const LE_GLOBAL float *)a.u)[((long long)s * a.m + t.t0 + i) * a.rank + j];
            lu[id] = f * v;
        }
        __syncthreads();
        float acc[16];
#pragma unroll
        for (int i = 0; i < 16; i++) acc[i] = 0.f;
        const long long row = ((long long)t.cur * a.rows + rc) * a.rank;
        for (int j = 0; j < a.rank; j += 8) {
            const Eight<WTY> w = load8<WTY>(a.b, row + j, a.rank - j);
#pragma unroll
            for (int i = 0; i < 16; i++)
                if (t.members >> i & 1) {
                    const float *u = lu + i * rp + j;
#pragma unroll
                    for (int k = 0; k < 8; k++) acc[i] = fmaf(w.up(k), u[k], acc[i]);
                }
        }
        if (r < a.rows) {
#pragma unroll
            for (int i = 0; i < 16; i++)
                if (t.members >> i & 1) ((LE_GLOBAL X *)a.y)[(t.t0 + i) * a.ldy + r] = XT<XTY>::down(b[i] + acc[i]);
        }
    }
}

/* ---- up, many tokens ----
 * A wave 64 output rows by 16 tokens. Of the 16 x 16 results of a matrix instruction a lane has four rows of its token; which rows of B are
 * its operand is free, and they are dealt so that four instructions leave 16 consecutive outputs in a lane. */
template <int WTY> __device__ __forceinline__ void upm_body(const LoraArgs &a) {
    const int l = threadIdx.x & 63, g = l >> 4, c16 = l & 15, r0 = (blockIdx.x * 4 + (threadIdx.x >> 6)) * 64;
    if (r0 >= a.rows) return;
    Tile t(a, blockIdx.y);
    const int tok = t.t0 + c16, tc = min(tok, a.m - 1), mine = r0 + 16 * g;
    using v4u_any = Any<sizeof(X)>::v;
    constexpr int PIECES = sizeof(X), E = 16 / sizeof(X); /* 16-byte pieces of 16 outputs, values of each */
    float out[16];
    const LE_GLOBAL X *base = (const LE_GLOBAL X *)a.base + tc * a.ldb + mine;
#pragma unroll
    for (int i = 0; i < 16; i++) out[i] = 0.f;
    if (a.base) {
#pragma unroll
        for (int p = 0; p < PIECES; p++) {
            if (mine + 16 <= a.rows) {
                const v4u v = *(const LE_GLOBAL v4u_any *)(base + p * E);
#pragma unroll
                for (int e = 0; e < E; e++) out[p * E + e] = unpack<XTY>(v, e);
            } else {
#pragma unroll
                for (int e = 0; e < E; e++)
                    if (mine + p * E + e < a.rows) out[p * E + e] = XT<XTY>::up(base[p * E + e]);
            }
        }
    }
    while (t.next()) {
        v4f c[4];
        long long brow[4];
#pragma unroll
        for (int f = 0; f < 4; f++) {
            c[f] = v4f{0.f, 0.f, 0.f, 0.f};
            brow[f] = ((long long)t.cur * a.rows + min(r0 + (c16 >> 2) * 16 + f * 4 + (c16 & 3), a.rows - 1)) * a.rank;
        }
        const float s = factor(a, t.cur);
        for (int j = 8 * g; j - 8 * g < a.rank; j += 32) {
            Eight<0> u;
#pragma unroll
            for (int i = 0; i < 8; i++) u.v[i] = 0.f;
            if (t.id == t.cur)
                for (int seg = 0; seg < a.segs; seg++) {
                    const Eight<0> p = load8<0>(a.u, ((long long)seg * a.m + tok) * a.rank + j, a.rank - j);
#pragma unroll
                    for (int i = 0; i < 8; i++) u.v[i] += p.v[i];
                }
#pragma unroll
            for (int i = 0; i < 8; i++) u.v[i] *= s;
#pragma unroll
            for (int f = 0; f < 4; f++) c[f] = multiply<WTY, 0>(load8<WTY>(a.b, brow[f] + j, a.rank - j), u, c[f]);
        }
        if (t.id == t.cur) {
#pragma unroll
            for (int f = 0; f < 4; f++)
#pragma unroll
                for (int i = 0; i < 4; i++) out[4 * f + i] += c[f][i];
        }
    }
    if (tok >= a.m) return;
    LE_GLOBAL X *y = (LE_GLOBAL X *)a.y + tok * a.ldy + mine;
#pragma unroll
    for (int p = 0; p < PIECES; p++) {
        if (mine + 16 <= a.rows) {
            v4u v;
#pragma unroll
            for (int d = 0; d < 4; d++) v[d] = pack<XTY>(out + p * E, d);
            *(LE_GLOBAL v4u_any *)(y + p * E) = v;
        } else {
#pragma unroll
            for (int e = 0; e < E; e++)
                if (mine + p * E + e < a.rows) y[p * E + e] = XT<XTY>::down(out[p * E + e]);
        }
    }
}

}  // namespace

#define LE_LO_NAME2(WHAT, X, W) le_lo_##WHAT##_##X##_##W
#define LE_LO_NAME(WHAT, X, W) LE_LO_NAME2(WHAT, X, W)
#define LE_LO(W)                                                                                                              \
    extern "C" __global__ void __launch_bounds__(256) LE_LO_NAME(down1, LE_LO_XTY, W)(LoraArgs a) { down_body<W, 1>(a); } \
    extern "C" __global__ void __launch_bounds__(256) LE_LO_NAME(down2, LE_LO_XTY, W)(LoraArgs a) { down_body<W, 2>(a); } \
    extern "C" __global__ void __launch_bounds__(256) LE_LO_NAME(down4, LE_LO_XTY, W)(LoraArgs a) { down_body<W, 4>(a); } \
    extern "C" __global__ void __launch_bounds__(256) LE_LO_NAME(upv, LE_LO_XTY, W)(LoraArgs a) { upv_body<W>(a); }       \
    extern "C" __global__ void __launch_bounds__(256) LE_LO_NAME(upm, LE_LO_XTY, W)(LoraArgs a) { upm_body<W>(a); }
LE_LO(0)
LE_LO(1)
LE_LO(30)
