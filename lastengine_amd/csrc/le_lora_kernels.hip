/* Low-rank adapters beside a shared projection (le_lora, include/le_qmm.h), compiled once per type of the activations (LE_LO_XTY).
 * Two launches: u[t] = A x[t] over the columns, then y[t] = base[t] + scale (B u[t]) over the rank. Tokens are taken 16 at a time, as they
 * come; a tile of 16 with several adapters is done once for each of them, and what it gives for the others' tokens is dropped
 * (selected, so that nothing of one token or adapter reaches another). */
#include <hip/hip_runtime.h>

#include "le_f32_types.h"
#include "le_lanes.h"
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

/* The eight values from p on, or zeros. */
template <int TY> __device__ __forceinline__ Eight<TY> whole8(const void *base, long long at, bool there) {
    using T = typename XT<TY>::raw;
    const LE_GLOBAL T *p = (const LE_GLOBAL T *)base + at;
    v4u lo = {0, 0, 0, 0}, hi = {0, 0, 0, 0};
    if (there) {
        lo = *(const LE_GLOBAL typename Any<sizeof(T)>::v *)p;
        if constexpr (TY == 0) hi = *(const LE_GLOBAL typename Any<sizeof(T)>::v *)(p + 4);
    }
    Eight<TY> r;
    if constexpr (TY == 0) {
        *(v4u *)&r.v[0] = lo;
        *(v4u *)&r.v[4] = hi;
    } else {
        r.v = lo;
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

/* ---- products ----
 * An operand of a matrix instruction over 32 of k: 16 rows, a lane's row l % 16 and its eight k from 8 (l / 16) on. Two operands of one 16-bit
 * type multiply as they are. Otherwise values are cut into bf16 pieces that add up to them exactly (fp16: 2 of 8 bits or less, fp32: 3 of 8,
 * cut off, not rounded) and every piece of one multiplies every piece of the other: two to five times faster than fp32 instructions, which are left for two
 * fp32 operands. Either way the products are exact (fp32: a fused multiply-add's) and the sums fp32. */
template <int TY, bool CUT> struct Operand;
template <int TY> struct Operand<TY, false> {
    Eight<TY> p[1];
    static constexpr int N = 1;
    __device__ __forceinline__ void set(const Eight<TY> &e) { p[0] = e; }
};
template <int TY> struct Operand<TY, true> {
    static constexpr int N = TY == 0 ? 3 : 2;
    v4u p[N];
    __device__ __forceinline__ void set(const Eight<TY> &e) {
        float v[8];
#pragma unroll
        for (int i = 0; i < 8; i++) v[i] = e.up(i);
#pragma unroll
        for (int n = 0; n < N; n++)
#pragma unroll
            for (int d = 0; d < 4; d++) {
                const unsigned lo = __builtin_bit_cast(unsigned, v[2 * d]), hi = __builtin_bit_cast(unsigned, v[2 * d + 1]);
                p[n][d] = __builtin_amdgcn_perm(hi, lo, 0x07060302);
                if (n + 1 < N) {
                    v[2 * d] -= __builtin_bit_cast(float, lo & 0xFFFF0000u);
                    v[2 * d + 1] -= __builtin_bit_cast(float, hi & 0xFFFF0000u);
                }
            }
    }
};
/* The first operand's form and the second's, for types P and Q. */
template <int P, int Q> struct Pair {
    static constexpr bool same = P == Q;
    using A = Operand<P, !same && P != 30>;
    using B = Operand<Q, !same && Q != 30>;
};
__device__ __forceinline__ v4u raw(const v4u &v) { return v; }
template <int TY> __device__ __forceinline__ v4u raw(const Eight<TY> &v) { return v.v; }
template <int P, int Q> __device__ __forceinline__ v4f multiply(const typename Pair<P, Q>::A &a, const typename Pair<P, Q>::B &b, v4f c) {
    if constexpr (P == 0 && Q == 0) {
#pragma unroll
        for (int i = 0; i < 8; i++) c = __builtin_amdgcn_mfma_f32_16x16x4f32(a.p[0].v[i], b.p[0].v[i], c, 0, 0, 0);
    } else if constexpr (P == 1 && Q == 1) {
        c = __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(v8h, a.p[0].v), __builtin_bit_cast(v8h, b.p[0].v), c, 0, 0, 0);
    } else {
#pragma unroll
        for (int i = 0; i < Pair<P, Q>::A::N; i++)
#pragma unroll
            for (int j = 0; j < Pair<P, Q>::B::N; j++)
                c = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(v8b, raw(a.p[i])), __builtin_bit_cast(v8b, raw(b.p[j])), c, 0, 0, 0);
    }
    return c;
}

/* ---- the adapters of a tile ---- */

/* Adapter of token t; -1: none, or no token */
__device__ __forceinline__ int adapter(const LoraArgs &a, int t) {
    const int id = t < a.m ? ((const LE_GLOBAL int *)a.idx)[t] : -1;
    return id < a.n_ad && id >= 0 ? id : -1;
}
struct Tile {
    int id;           /* adapter of this lane's token, its lane % 16th of the tile */
    unsigned left;    /* tokens whose adapter has not come yet */
    int cur;
    unsigned members; /* tokens of adapter cur */
    __device__ __forceinline__ Tile(int id) : id(id), left((unsigned)__ballot(id >= 0) & 0xFFFF) {}
    __device__ __forceinline__ bool next() {
        if (!left) return false;
        cur = __builtin_amdgcn_readlane(id, __ffs((int)left) - 1);
        members = (unsigned)__ballot(id == cur) & 0xFFFF;
        left &= ~members;
        return true;
    }
};

/* Where u of token i of a tile has rank j: in the order of a matrix instruction's operand (32 ranks of 16 tokens, two pieces of 16 bytes a lane), so
 * that a wave reads whole lines; ranks are filled up with zeros to a multiple of 32. */
__device__ __forceinline__ long long place(const LoraArgs &a, int seg, int tile, int i, int j) {
    const int jb = (a.rank + 31) >> 5, lane = i + 16 * (j >> 3 & 3);
    return ((((long long)seg * ((a.m + 15) >> 4) + tile) * jb + (j >> 5)) * 2 + (j >> 2 & 1)) * 256 + lane * 4 + (j & 3);
}

/* ---- down: u = A x ----
 * A block takes a tile, an adapter of it and a segment of the columns, its waves 64 columns in turn; their sums meet in LDS. Rows of A
 * as the other operand, RF times 16 of them at once. A wave reads 128 (fp32: 256) bytes of a row at a time, in whole lines, and turns them to
 * the matrix instruction's layout through LDS of its own (read in that layout from memory, 16 bytes in each of 16 rows side by side, the same
 * kernel took twice the time), the next step's on their way meanwhile. */
template <int TY> struct Rows { /* 16 rows of 64 values */
    static constexpr int V = TY == 0 ? 4 : 8, LANES = 64 / V, N = 16 * LANES / 64, PITCH = 64 * (16 / V) + 16;
    static constexpr int BYTES = 16 * PITCH;
    v4u r[N];
    __device__ __forceinline__ void load(const void *base, const long long *row, int k, bool whole, int cols) {
        using T = typename XT<TY>::raw;
        const int l = threadIdx.x & 63, at = k + l % LANES * V;
#pragma unroll
        for (int n = 0; n < N; n++) {
            const LE_GLOBAL T *p = (const LE_GLOBAL T *)base + row[n] + at;
            if (whole || at + V <= cols) {
                r[n] = *(const LE_GLOBAL typename Any<sizeof(T)>::v *)p;
            } else {
                r[n] = v4u{0, 0, 0, 0};
#pragma unroll
                for (int e = 0; e < V; e++)
                    if (at + e < cols) {
                        const typename XT<TY>::raw v = p[e];
                        if constexpr (V == 4) r[n][e] = __builtin_bit_cast(unsigned, v);
                        else r[n][e >> 1] |= (unsigned)v << (e & 1) * 16;
                    }
            }
        }
    }
    __device__ __forceinline__ void store(char *lds) const {
        const int l = threadIdx.x & 63;
#pragma unroll
        for (int n = 0; n < N; n++) *(v4u *)(lds + (n * (64 / LANES) + l / LANES) * PITCH + l % LANES * 16) = r[n];
    }
    static __device__ __forceinline__ int row_of(int n) { return n * (64 / LANES) + (threadIdx.x & 63) / LANES; }
    static __device__ __forceinline__ Eight<TY> read(const char *lds, int half) {
        const int l = threadIdx.x & 63;
        const char *p = lds + (l & 15) * PITCH + (32 * half + 8 * (l >> 4)) * (16 / V);
        Eight<TY> e;
        if constexpr (TY == 0) {
            *(v4f *)&e.v[0] = *(const v4f *)p;
            *(v4f *)&e.v[4] = *(const v4f *)(p + 16);
        } else {
            e.v = *(const v4u *)p;
        }
        return e;
    }
};
template <int WTY, int RF> __device__ __forceinline__ void down_body(const LoraArgs &a) {
    using Mul = Pair<XTY, WTY>;
    using XR = Rows<XTY>;
    using WR = Rows<WTY>;
    extern __shared__ __attribute__((aligned(16))) char lds[]; /* each wave's rows, then its sums: [wave][RF][256] */
    const int l = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), nw = blockDim.x >> 6;
    const int tile = blockIdx.x, turn = blockIdx.y, turns = gridDim.y, t0 = tile * 16;
    char *mine = lds + wave * (XR::BYTES + RF * WR::BYTES);
    Tile t(adapter(a, t0 + (l & 15)));
    const int s0 = blockIdx.z * a.steps + wave, s1 = min((int)(blockIdx.z + 1) * a.steps, (a.cols + 63) / 64);
    long long xrow[XR::N];
#pragma unroll
    for (int n = 0; n < XR::N; n++) xrow[n] = min(t0 + XR::row_of(n), a.m - 1) * a.ldx;
    for (int nth = 0; t.next(); nth++) {
        if (nth % turns != turn) continue;
        for (int j0 = 0; j0 < a.rank; j0 += 16 * RF) {
            v4f c[RF];
            long long arow[RF][WR::N];
#pragma unroll
            for (int f = 0; f < RF; f++) {
                c[f] = v4f{0.f, 0.f, 0.f, 0.f};
#pragma unroll
                for (int n = 0; n < WR::N; n++) arow[f][n] = ((long long)t.cur * a.rank + min(j0 + 16 * f + WR::row_of(n), a.rank - 1)) * a.cols;
            }
            XR x;
            WR w[RF];
            auto load = [&](int s) {
                const bool whole = 64 * s + 64 <= a.cols;
                x.load(a.x, xrow, 64 * s, whole, a.cols);
#pragma unroll
                for (int f = 0; f < RF; f++) w[f].load(a.a, arow[f], 64 * s, whole, a.cols);
            };
            if (s0 < s1) load(s0);
            for (int s = s0; s < s1; s += nw) {
                __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront"); /* the reads of the step before */
                __builtin_amdgcn_wave_barrier();
                x.store(mine);
#pragma unroll
                for (int f = 0; f < RF; f++) w[f].store(mine + XR::BYTES + f * WR::BYTES);
                if (s + nw < s1) load(s + nw);
                __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
                __builtin_amdgcn_wave_barrier();
#pragma unroll
                for (int half = 0; half < 2; half++) {
                    typename Mul::A p;
                    p.set(XR::read(mine, half));
#pragma unroll
                    for (int f = 0; f < RF; f++) {
                        typename Mul::B q;
                        q.set(WR::read(mine + XR::BYTES + f * WR::BYTES, half));
                        c[f] = multiply<XTY, WTY>(p, q, c[f]);
                    }
                }
            }
            float *sums = (float *)lds;
            __syncthreads();
#pragma unroll
            for (int f = 0; f < RF; f++)
#pragma unroll
                for (int e = 0; e < 4; e++) sums[(wave * RF + f) * 256 + ((l >> 4) * 4 + e) * 16 + (l & 15)] = c[f][e];
            __syncthreads();
            for (int id = threadIdx.x; id < 256 * RF; id += blockDim.x) {
                const int row = id >> 4 & 15, j = j0 + (id >> 8) * 16 + (id & 15);
                if (j < ((a.rank + 31) & ~31) && (t.members >> row & 1)) {
                    float v = sums[id];
                    for (int n = 1; n < nw; n++) v += sums[n * RF * 256 + id];
                    ((LE_GLOBAL float *)a.u)[place(a, blockIdx.z, tile, row, j)] = j < a.rank ? v : 0.f;
                    if (RF == 1) ((LE_GLOBAL float *)a.u)[place(a, blockIdx.z, tile, row, j + 16)] = 0.f; /* rank <= 16 here */
                }
            }
            __syncthreads();
        }
    }
}

__device__ __forceinline__ float factor(const LoraArgs &a, int ad) { return a.scale ? ((const LE_GLOBAL float *)a.scale)[ad] : 1.f; }

/* ---- up, few tokens ----
 * A wave 64 output rows, G lanes with eight values each a row of B (so that a wave's loads are whole lines), G turns for all of them; after
 * each the group's sum stays with the lane whose row it is. Lane l ends with row l. B is read once for all tokens of the adapter up to
 * a rank of 64, and the tokens are taken four at a time. u of the whole tile is fetched beside the adapters' numbers, not after them, and
 * the next 64 rows' operands during these' sums (above a rank of 64 B does not fit and is fetched for every four tokens). */
template <int WTY, int G> __device__ __forceinline__ void upv_body(const LoraArgs &a) {
    constexpr int RP = 8 * G, TURNS = G < 8 ? G : 8; /* turns whose B is in registers at once */
    __shared__ __attribute__((aligned(16))) float lu[16][RP]; /* A x of the tile's tokens; of those without an adapter nothing that is used */
    const int l = threadIdx.x & 63, t0 = blockIdx.y * 16;
    const int id = adapter(a, t0 + (l & 15));
    const long long seg = place(a, 1, 0, 0, 0);
    for (int i = threadIdx.x; i < 16 * RP; i += 256) {
        const int j = i & (RP - 1);
        const LE_GLOBAL float *u = (const LE_GLOBAL float *)a.u + place(a, 0, blockIdx.y, i / RP, j);
        float v = 0.f;
        if (j < a.rank)
#pragma unroll 8
            for (int s = 0; s < a.segs; s++) v += u[s * seg];
        lu[0][i] = v;
    }
    __syncthreads();
    Tile t(id);
    const LE_GLOBAL X *base = (const LE_GLOBAL X *)a.base;
    LE_GLOBAL X *y = (LE_GLOBAL X *)a.y;
    const int step = gridDim.x * 256, first = (blockIdx.x * 4 + (threadIdx.x >> 6)) * 64, part = l & (G - 1);
    if (blockIdx.z == 0) { /* tokens of no adapter */
        for (unsigned none = ~t.left & 0xFFFF; none; none &= none - 1) {
            const int k = t0 + __ffs((int)none) - 1;
            if (k >= a.m) break;
            for (int r = first + l; r < a.rows; r += step) y[k * a.ldy + r] = a.base ? base[k * a.ldb + r] : X(0);
        }
    }
    for (int nth = 0; t.next(); nth++) {
        if (nth % gridDim.z != blockIdx.z) continue;
        struct Four {
            int k[4]; /* tokens; the last one again where fewer are left */
            __device__ __forceinline__ Four(unsigned &todo) {
#pragma unroll
                for (int i = 0; i < 4; i++) {
                    k[i] = todo ? __ffs((int)todo) - 1 : k[i > 0 ? i - 1 : 0];
                    todo &= todo - 1;
                }
            }
            __device__ __forceinline__ bool is(int i) const { return i == 0 || k[i] != k[i - 1]; }
        };
        struct Ahead { /* what the first four tokens' results of 64 rows are made of */
            Eight<WTY> w[TURNS];
            float b[4];
        } now, next;
        auto load = [&](Eight<WTY> *w, int r0, int turn) {
#pragma unroll
            for (int p = 0; p < TURNS; p++)
                w[p] = load8<WTY>(a.b, ((long long)t.cur * a.rows + min(r0 + l - part + turn + p, a.rows - 1)) * a.rank + 8 * part, a.rank - 8 * part);
        };
        auto bases = [&](const Four &q, float *b, int r0) {
#pragma unroll
            for (int i = 0; i < 4; i++) {
                b[i] = 0.f;
                if (a.base && q.is(i)) b[i] = XT<XTY>::up(base[(t0 + q.k[i]) * a.ldb + min(r0 + l, a.rows - 1)]);
            }
        };
        unsigned others = t.members;
        const Four four(others);
        if (first < a.rows) load(now.w, first, 0), bases(four, now.b, first);
        const float f = factor(a, t.cur);
        for (int r0 = first; r0 < a.rows; r0 += step, now = next) {
            if (r0 + step < a.rows) load(next.w, r0 + step, 0), bases(four, next.b, r0 + step);
            auto take = [&](const Four &q, const float *b) {
                float acc[4], u[4][8];
#pragma unroll
                for (int i = 0; i < 4; i++) {
                    acc[i] = 0.f;
                    if (q.is(i)) {
                        *(v4f *)&u[i][0] = *(const v4f *)&lu[q.k[i]][8 * part];
                        *(v4f *)&u[i][4] = *(const v4f *)&lu[q.k[i]][8 * part + 4];
                    }
                }
#pragma unroll 1
                for (int turn = 0; turn < G; turn += TURNS) {
                    if (G > 8) load(now.w, r0, turn);
#pragma unroll
                    for (int i = 0; i < 4; i++)
                        if (q.is(i)) {
#pragma unroll
                            for (int p = 0; p < TURNS; p++) {
                                float s = now.w[p].up(0) * u[i][0];
#pragma unroll
                                for (int e = 1; e < 8; e++) s = fmaf(now.w[p].up(e), u[i][e], s);
                                s = lanes_sum<G>(s);
                                if (part == turn + p) acc[i] = s;
                            }
                        }
                }
#pragma unroll
                for (int i = 0; i < 4; i++)
                    if (q.is(i) && r0 + l < a.rows) y[(t0 + q.k[i]) * a.ldy + r0 + l] = XT<XTY>::down(fmaf(f, acc[i], b[i]));
            };
            take(four, now.b);
            for (unsigned todo = others; todo;) {
                const Four q(todo);
                float b[4];
                bases(q, b, r0);
                take(q, b);
            }
        }
    }
}

/* ---- up, many tokens ----
 * A wave 64 output rows by up to 64 tokens, 16 at a time. A matrix instruction leaves four rows of 16 tokens in a lane; they change places through LDS, so
 * that base is read and y written in whole rows of 64 (128 or 256 bytes). B stays in registers while the adapter does, for ranks that are
 * multiples of 8 up to 32 J (J = 0, any other rank: read for each tile). */
template <int WTY, int J> __device__ __forceinline__ void upm_body(const LoraArgs &a) {
    using v4u_any = Any<sizeof(X)>::v;
    using Mul = Pair<WTY, 0>;
    constexpr int E = 16 / sizeof(X), LANES = 64 / E, PIECES = 16 / E; /* values of a piece, lanes of a row of 64, pieces of a lane */
    constexpr int PITCH = 68;
    __shared__ __attribute__((aligned(16))) float turn[4][16 * PITCH];
    float *mine = turn[threadIdx.x >> 6];
    const int l = threadIdx.x & 63, g = l >> 4, c16 = l & 15, r0 = (blockIdx.x * 4 + (threadIdx.x >> 6)) * 64;
    if (r0 >= a.rows) return;
    const int row = r0 + l % LANES * E; /* first of this lane's piece */
    const bool whole = row + E <= a.rows;
    const int ids = adapter(a, blockIdx.y * 64 + l);
    int held = -1; /* whose B the registers hold */
    const float none = a.base ? -0.f : 0.f; /* a token's factor without an adapter: what its zeros then add leaves base as it is, a zero of either sign too
                                             * (sums that begin at that instead of 0 take 44 registers more) */
    typename Mul::A w[J > 0 ? J : 1][4];
    auto get = [&](int ad, int j, typename Mul::A *q) {
#pragma unroll
        for (int f = 0; f < 4; f++) {
            const long long at = ((long long)ad * a.rows + min(r0 + 16 * f + c16, a.rows - 1)) * a.rank + j + 8 * g;
            if constexpr (J == 0) q[f].set(load8<WTY>(a.b, at, a.rank - j - 8 * g));
            else q[f].set(whole8<WTY>(a.b, at, j + 8 * g < a.rank));
        }
    };
#pragma unroll
    for (int n = 0; n < 4; n++) {
        const int t0 = blockIdx.y * 64 + 16 * n, tok = t0 + c16;
        if (t0 >= a.m) break;
        v4u base[PIECES];
#pragma unroll
        for (int p = 0; p < PIECES; p++)
            if (a.base && whole) base[p] = *(const LE_GLOBAL v4u_any *)((const LE_GLOBAL X *)a.base + min(t0 + p * E + l / LANES, a.m - 1) * a.ldb + row);
        Tile t(__builtin_amdgcn_ds_bpermute((16 * n + c16) * 4, ids));
        const float s = t.id >= 0 ? factor(a, t.id) : none;
        /* u of this lane's token, zeros where it has no adapter */
        auto low = [&](int j) {
            Eight<0> u;
#pragma unroll
            for (int i = 0; i < 8; i++) u.v[i] = 0.f;
            if (t.id >= 0)
                for (int seg = 0; seg < a.segs; seg++) {
                    const LE_GLOBAL float *from = (const LE_GLOBAL float *)a.u + place(a, seg, t0 >> 4, c16, j + 8 * g);
                    const v4f lo = *(const LE_GLOBAL v4f *)from, hi = *(const LE_GLOBAL v4f *)(from + 256);
#pragma unroll
                    for (int i = 0; i < 4; i++) u.v[i] += lo[i], u.v[4 + i] += hi[i];
                }
            return u;
        };
        typename Mul::B u[J > 0 ? J : 1];
        if constexpr (J > 0) {
#pragma unroll
            for (int j = 0; j < J; j++) u[j].set(low(32 * j));
        }
        v4f out[4];
#pragma unroll
        for (int f = 0; f < 4; f++) out[f] = v4f{0.f, 0.f, 0.f, 0.f};
        while (t.next()) {
            v4f c[4];
#pragma unroll
            for (int f = 0; f < 4; f++) c[f] = v4f{0.f, 0.f, 0.f, 0.f};
            if constexpr (J > 0) {
                if (t.cur != held) {
#pragma unroll
                    for (int j = 0; j < J; j++) get(t.cur, 32 * j, w[j]);
                    held = t.cur;
                }
#pragma unroll
                for (int j = 0; j < J; j++)
#pragma unroll
                    for (int f = 0; f < 4; f++) c[f] = multiply<WTY, 0>(w[j][f], u[j], c[f]);
            } else {
                for (int j = 0; j < a.rank; j += 32) {
                    u[0].set(low(j));
                    get(t.cur, j, w[0]);
#pragma unroll
                    for (int f = 0; f < 4; f++) c[f] = multiply<WTY, 0>(w[0][f], u[0], c[f]);
                }
            }
            if (t.id == t.cur) {
#pragma unroll
                for (int f = 0; f < 4; f++) out[f] = c[f];
            }
        }
#pragma unroll
        for (int f = 0; f < 4; f++) out[f] *= s; /* behind the sum, as for few tokens: scale u may be out of fp32's range where y is not */
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront"); /* the wave's reads of the tile before */
        __builtin_amdgcn_wave_barrier();
#pragma unroll
        for (int f = 0; f < 4; f++) *(v4f *)&mine[c16 * PITCH + 16 * f + 4 * g] = out[f];
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        __builtin_amdgcn_wave_barrier();
#pragma unroll
        for (int p = 0; p < PIECES; p++) {
            const int i = p * E + l / LANES, k = t0 + i;
            float v[E];
#pragma unroll
            for (int e = 0; e < E; e += 4) *(v4f *)&v[e] = *(const v4f *)&mine[i * PITCH + l % LANES * E + e];
            if (k >= a.m) continue;
            LE_GLOBAL X *y = (LE_GLOBAL X *)a.y + k * a.ldy + row;
            if (whole) {
                if (a.base) {
#pragma unroll
                    for (int e = 0; e < E; e++) v[e] += unpack<XTY>(base[p], e);
                }
                v4u q;
#pragma unroll
                for (int d = 0; d < 4; d++) q[d] = pack<XTY>(v, d);
                *(LE_GLOBAL v4u_any *)y = q;
            } else {
#pragma unroll
                for (int e = 0; e < E; e++)
                    if (row + e < a.rows) y[e] = XT<XTY>::down(a.base ? XT<XTY>::up(((const LE_GLOBAL X *)a.base)[k * a.ldb + row + e]) + v[e] : v[e]);
            }
        }
    }
}

}  // namespace

#define LE_LO_NAME2(WHAT, X, W) le_lo_##WHAT##_##X##_##W
#define LE_LO_NAME(WHAT, X, W) LE_LO_NAME2(WHAT, X, W)
/* Waves a SIMD of upm0: four where 128 registers do without scratch (fp32 adapters of rank 37 beside fp16, 4096 tokens 59 us, with one register too many 66) */
#define LE_LO_FOUR(W) (LE_LO_XTY != 0 && W != 1 ? 4 : 3)
#define LE_LO(W)                                                                                                             \
    extern "C" __global__ void __launch_bounds__(512) LE_LO_NAME(down1, LE_LO_XTY, W)(LoraArgs a) { down_body<W, 1>(a); } \
    extern "C" __global__ void __launch_bounds__(512) LE_LO_NAME(down2, LE_LO_XTY, W)(LoraArgs a) { down_body<W, 2>(a); } \
    extern "C" __global__ void __launch_bounds__(512) LE_LO_NAME(down4, LE_LO_XTY, W)(LoraArgs a) { down_body<W, 4>(a); } \
    extern "C" __global__ void __launch_bounds__(256) LE_LO_NAME(upv1, LE_LO_XTY, W)(LoraArgs a) { upv_body<W, 1>(a); } \
    extern "C" __global__ void __launch_bounds__(256) LE_LO_NAME(upv2, LE_LO_XTY, W)(LoraArgs a) { upv_body<W, 2>(a); } \
    extern "C" __global__ void __launch_bounds__(256) LE_LO_NAME(upv4, LE_LO_XTY, W)(LoraArgs a) { upv_body<W, 4>(a); } \
    extern "C" __global__ void __launch_bounds__(256) LE_LO_NAME(upv8, LE_LO_XTY, W)(LoraArgs a) { upv_body<W, 8>(a); } \
    extern "C" __global__ void __launch_bounds__(256) LE_LO_NAME(upv16, LE_LO_XTY, W)(LoraArgs a) { upv_body<W, 16>(a); } \
    extern "C" __global__ void __launch_bounds__(256) LE_LO_NAME(upv32, LE_LO_XTY, W)(LoraArgs a) { upv_body<W, 32>(a); } \
    extern "C" __global__ void __launch_bounds__(256, LE_LO_FOUR(W)) LE_LO_NAME(upm0, LE_LO_XTY, W)(LoraArgs a) { upm_body<W, 0>(a); }    \
    extern "C" __global__ void __launch_bounds__(256) LE_LO_NAME(upm1, LE_LO_XTY, W)(LoraArgs a) { upm_body<W, 1>(a); }    \
    extern "C" __global__ void __launch_bounds__(256) LE_LO_NAME(upm2, LE_LO_XTY, W)(LoraArgs a) { upm_body<W, 2>(a); }
LE_LO(0)
LE_LO(1)
LE_LO(30)
