/* Products of the routed experts over dense weights and their gradients (le_mm_experts, include/le_qmm.h), compiled once per type of
 * the rows (LE_EX_TY).
 *
 * All three are C[m][n] = sum over k of A[m][k] B[n][k] within an expert:
 *   y:  m = the expert's rows, n = rows of W,  k = columns;  A = x,  B = W
 *   dx: m = the expert's rows, n = columns,    k = rows of W; A = dy, B = W read down its columns
 *   dw: m = rows of W, n = columns, k = the expert's rows;    A = dy, B = x, both read down their columns
 * An operand whose k lies along its rows in memory ("along") and one whose k counts its rows ("down") go to LDS as they lie, in 16-byte
 * chunks: a tile of `along` is [row][64 bytes of k], one of `down` [k][row]. Matrix instructions want 8 (fp32: 4) values of k a lane; from a
 * `down` tile the transposing LDS read of 16-bit values gives them, or for fp32 a 4-byte read each. Chunks are permuted within
 * their row (swizzle) so that the rows of one read lie in different banks. */
#include <hip/hip_runtime.h>

#include "le_experts_args.h"
#include "le_f32_types.h"

#define LE_GLOBAL __attribute__((address_space(1)))
#define LE_LDS __attribute__((address_space(3)))

namespace {

constexpr int TY = LE_EX_TY;
using T = XT<TY>::raw;
constexpr int ES = sizeof(T), EPC = 16 / ES; /* bytes a value, values a chunk */
constexpr int BK = 64 / ES;                  /* depth of a step */

typedef unsigned v4u __attribute__((ext_vector_type(4)));
typedef v4u __attribute__((aligned(ES))) v4u_any;
typedef float v4f __attribute__((ext_vector_type(4)));
typedef float v16f __attribute__((ext_vector_type(16)));
typedef short v4s __attribute__((ext_vector_type(4)));
typedef short v8s __attribute__((ext_vector_type(8)));
typedef _Float16 v8h __attribute__((ext_vector_type(8)));
typedef __bf16 v8b __attribute__((ext_vector_type(8)));

/* ---- tiles in LDS ---- */

template <bool DOWN, int R> __device__ __forceinline__ int lds_at(int row_or_k, int chunk) {
    if constexpr (!DOWN) return row_or_k * 64 + ((chunk ^ ((row_or_k >> 2) & 3)) << 4);
    constexpr int C = R / EPC; /* chunks a k */
    const int sw = ES == 2 ? (row_or_k & 3) << 2 : ((row_or_k >> 2) & 1) << 3;
    return row_or_k * (R * ES) + ((chunk ^ (sw & (C - 1))) << 4);
}

/* A lane's operand for half a step (fp32: of 8 values of k, else of 16): row row0 + lane % 32, k = (2 s + lane / 32) * EPC + 0 .. EPC - 1 */
union Frag {
    v4u u;
    v4f f;
    v8s s;
    struct {
        v4s lo, hi;
    } p;
};
template <bool DOWN, int R> __device__ __forceinline__ Frag frag(LE_LDS const char *tile, int row0, int s, int l) {
    Frag v;
    if constexpr (!DOWN) {
        v.u = *(LE_LDS const v4u *)(tile + lds_at<false, R>(row0 + (l & 31), 2 * s + (l >> 5)));
    } else if constexpr (ES == 4) {
        const int r = row0 + (l & 31), k = (2 * s + (l >> 5)) * 4;
#pragma unroll
        for (int j = 0; j < 4; j++) v.f[j] = *(LE_LDS const float *)(tile + lds_at<true, R>(k + j, r >> 2) + (r & 3) * 4);
    } else {
        /* 16 lanes read four k of 16 rows, 8 bytes each; lane i of them gets the four k of row i */
        const int i = l & 15, r = row0 + (l & 16) + (i & 3) * 4, k = (2 * s + (l >> 5)) * 8 + (i >> 2);
        typedef LE_LDS v4s *p4;
        v.p.lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((p4)(tile + lds_at<true, R>(k, r >> 3) + (r & 4) * 2));
        v.p.hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((p4)(tile + lds_at<true, R>(k + 4, r >> 3) + (r & 4) * 2));
    }
    return v;
}
__device__ __forceinline__ v16f mfma(const Frag &a, const Frag &b, v16f c) {
    if constexpr (TY == 0) {
#pragma unroll
        for (int j = 0; j < 4; j++) c = __builtin_amdgcn_mfma_f32_32x32x2f32(a.f[j], b.f[j], c, 0, 0, 0);
        return c;
    } else if constexpr (TY == 1) {
        return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(v8h, a.u), __builtin_bit_cast(v8h, b.u), c, 0, 0, 0);
    } else {
        return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(v8b, a.u), __builtin_bit_cast(v8b, b.u), c, 0, 0, 0);
    }
}

/* ---- which tile ---- */

struct Tile {
    int e, lo, cnt; /* expert, its first row, its rows */
    int m0, n0;
};
/* An expert's rows, within the buffers whatever off holds. */
__device__ __forceinline__ void rows_of(const ExpertArgs &a, int e, int &lo, int &cnt) {
    const LE_GLOBAL int *off = (const LE_GLOBAL int *)a.off;
    lo = min(max(off[e], 0), a.n_row);
    cnt = min(max(off[e + 1], lo), a.n_row) - lo;
}
/* Blocks go to the XCDs in turn: `run` consecutive tiles to each, so that tiles that share weights share an L2. */
__device__ __forceinline__ long long tile_of(const ExpertArgs &a, long long b) {
    const int turn = 8 * a.run, r = (int)(b % turn);
    return b - r + (r & 7) * a.run + (r >> 3);
}
/* Tile q of mt x nt, rows of tiles in groups of eight so that a group's rows and columns stay in the L2. */
template <int BM, int BN> __device__ __forceinline__ void place(Tile &t, long long q, int mt, int nt) {
    const int g = (int)(q / (8LL * nt)), r = (int)(q - 8LL * nt * g), gm = min(8, mt - 8 * g);
    t.n0 = r / gm * BN;
    t.m0 = (8 * g + r % gm) * BM;
}
/* Tile t of an expert's rows by outputs; every wave finds it by itself, 64 experts a turn. False: behind the last. */
template <int BM, int BN> __device__ __forceinline__ bool find_rows(const ExpertArgs &a, long long q, Tile &t) {
    const int l = threadIdx.x & 63, u = (int)(q / a.nt); /* row tiles before this one, over all experts */
    int before = 0;
    for (int e0 = 0; e0 < a.n_exp; e0 += 64) {
        int lo = 0, cnt = 0;
        if (e0 + l < a.n_exp) rows_of(a, e0 + l, lo, cnt);
        const int mine = (int)(((long long)cnt + BM - 1) / BM);
        int sum = mine;
#pragma unroll
        for (int d = 1; d < 64; d <<= 1) {
            const int v = __shfl_up(sum, d);
            if (l >= d) sum += v;
        }
        const unsigned long long hit = __ballot(u < before + sum);
        if (hit) {
            const int i = __ffsll((long long)hit) - 1;
            t.e = e0 + i;
            t.lo = __builtin_amdgcn_readlane(lo, i);
            t.cnt = __builtin_amdgcn_readlane(cnt, i);
            const int first = before + __builtin_amdgcn_readlane(sum - mine, i);
            place<BM, BN>(t, q - (long long)first * a.nt, (t.cnt + BM - 1) / BM, a.nt);
            return true;
        }
        before += __builtin_amdgcn_readlane(sum, 63);
    }
    return false;
}
template <int BM, int BN> __device__ __forceinline__ bool find_weights(const ExpertArgs &a, long long q, Tile &t) {
    const long long per = (long long)a.mt * a.nt;
    if (q >= per * a.n_exp) return false;
    t.e = (int)(q / per);
    rows_of(a, t.e, t.lo, t.cnt);
    place<BM, BN>(t, q - per * t.e, a.mt, a.nt);
    return true;
}

/* ---- any size, stride and alignment ----
 * 128 x 128 tiles by four waves of 128 x 32, chunks through registers (a 16-byte load at any address, values one by one at a row's end, zeros
 * beyond), the next step's in flight during this one's products. */

/* Up to EPC values from p, zeros behind the n that there are. */
__device__ __forceinline__ v4u load_chunk(const T *p, int n) {
    const LE_GLOBAL T *g = (const LE_GLOBAL T *)p;
    if (n >= EPC) return *(const LE_GLOBAL v4u_any *)g;
    v4u v = {0, 0, 0, 0};
#pragma unroll
    for (int j = 0; j < EPC - 1; j++)
        if (j < n) {
            if constexpr (ES == 4) v[j] = ((const LE_GLOBAL unsigned *)g)[j];
            else v[j >> 1] |= (unsigned)g[j] << (j & 1) * 16;
        }
    return v;
}
/* Chunks of R rows of an operand; `rows` of them there are, `depth` values of k. */
template <bool DOWN, int R> struct Loader {
    static constexpr int N = R * 64 / 16 / 256; /* chunks a thread */
    const T *base;
    long long ld;
    int rows, depth;
    v4u v[N];
    __device__ __forceinline__ void load(int k0) {
#pragma unroll
        for (int j = 0; j < N; j++) {
            const int id = threadIdx.x + 256 * j;
            if constexpr (!DOWN) {
                const int r = id >> 2, k = k0 + (id & 3) * EPC;
                v[j] = load_chunk(base + r * ld + k, r < rows ? depth - k : 0);
            } else {
                const int k = k0 + id / (R / EPC), r = id % (R / EPC) * EPC;
                v[j] = load_chunk(base + k * ld + r, k < depth ? rows - r : 0);
            }
        }
    }
    __device__ __forceinline__ void store(LE_LDS char *tile) const {
#pragma unroll
        for (int j = 0; j < N; j++) {
            const int id = threadIdx.x + 256 * j;
            const int at = !DOWN ? lds_at<false, R>(id >> 2, id & 3) : lds_at<true, R>(id / (R / EPC), id % (R / EPC));
            *(LE_LDS v4u *)(tile + at) = v[j];
        }
    }
};

enum Kind { Y, DX, DW };
template <int N> struct Count { static constexpr int value = N; };

/* ---- results ----
 * The operands go into the matrix instruction as (B, A): a lane then holds row l % 32 of the tile's 32 and 16 of 32 columns, four in a row. NF such
 * fragments side by side are rounded and change places through LDS of the wave's own, so that whole lines are written. */
template <int YTY, int NF> struct Out {
    using U = typename XT<YTY>::raw;
    static constexpr int E = 16 / sizeof(U), LANES = 32 * NF / E, PITCH = 32 * NF * sizeof(U) + 16, BYTES = 32 * PITCH;
    /* rows of them there are, at y, ld apart; cols of them there are, from this wave's first on */
    static __device__ __forceinline__ void put(LE_LDS char *mine, const v16f *c, void *y, long long ld, int rows, int cols) {
        typedef v4u __attribute__((aligned(4))) v4u_a4;
        typedef v4u __attribute__((aligned(2))) v4u_a2;
        const int l = threadIdx.x & 63;
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront"); /* the reads of the rows before */
        __builtin_amdgcn_wave_barrier();
#pragma unroll
        for (int n = 0; n < NF; n++)
#pragma unroll
            for (int q = 0; q < 4; q++) { /* columns 8 q + 4 (l / 32) and on */
                LE_LDS char *p = mine + (l & 31) * PITCH + (32 * n + 8 * q + 4 * (l >> 5)) * (int)sizeof(U);
                const float v0 = c[n][4 * q], v1 = c[n][4 * q + 1], v2 = c[n][4 * q + 2], v3 = c[n][4 * q + 3];
                if constexpr (sizeof(U) == 4) {
                    *(LE_LDS v4f *)p = v4f{v0, v1, v2, v3};
                } else {
                    typedef unsigned v2u __attribute__((ext_vector_type(2)));
                    *(LE_LDS v2u *)p = v2u{XT<YTY>::down(v0) | (unsigned)XT<YTY>::down(v1) << 16, XT<YTY>::down(v2) | (unsigned)XT<YTY>::down(v3) << 16};
                }
            }
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        __builtin_amdgcn_wave_barrier();
        const int col = l % LANES * E;
#pragma unroll
        for (int i = 0; i < 32; i += 64 / LANES) {
            const int r = i + l / LANES;
            const v4u v = *(LE_LDS const v4u *)(mine + r * PITCH + col * (int)sizeof(U));
            LE_GLOBAL U *to = (LE_GLOBAL U *)y + r * ld + col;
            if (r < rows) {
                if (col + E <= cols) {
                    if constexpr (sizeof(U) == 4) *(LE_GLOBAL v4u_a4 *)to = v;
                    else *(LE_GLOBAL v4u_a2 *)to = v;
                } else {
#pragma unroll
                    for (int e = 0; e < E - 1; e++)
                        if (col + e < cols) {
                            const unsigned w = v[sizeof(U) == 4 ? e : e >> 1];
                            if constexpr (sizeof(U) == 4) to[e] = __builtin_bit_cast(float, w);
                            else to[e] = (U)(w >> (e & 1) * 16);
                        }
                }
            }
        }
    }
};

template <Kind KIND, int YTY> __device__ __forceinline__ void any_body(const ExpertArgs &a) {
    constexpr int BM = 128, BN = 128, MF = BM / 32;
    constexpr bool AD = KIND == DW, BD = KIND != Y;
    constexpr int TILES = (BM + BN) * 64, OUT = 4 * Out<YTY, 1>::BYTES;
    __shared__ __attribute__((aligned(16))) char smem[TILES > OUT ? TILES : OUT];
    LE_LDS char *ta = (LE_LDS char *)smem, *tb = ta + BM * 64;
    const int l = threadIdx.x & 63, wn = (threadIdx.x >> 6) * 32;
    for (long long b = blockIdx.x;; b += gridDim.x) {
        Tile t;
        if (!(KIND == DW ? find_weights<BM, BN>(a, tile_of(a, b), t) : find_rows<BM, BN>(a, tile_of(a, b), t))) return;
        const int m = KIND == DW ? a.m : t.cnt, k = KIND == DW ? t.cnt : a.k;
        const long long wsize = KIND == Y ? (long long)a.n * a.k : (long long)a.k * a.n;
        Loader<AD, BM> A;
        Loader<BD, BN> B;
        A.ld = a.lda, A.rows = m - t.m0, A.depth = k;
        A.base = (const T *)a.a + (KIND == DW ? t.lo * a.lda + t.m0 : (long long)(t.lo + t.m0) * a.lda);
        B.ld = a.ldb, B.rows = a.n - t.n0, B.depth = k;
        B.base = (const T *)a.b + (KIND == DW ? t.lo * a.ldb + t.n0 : KIND == Y ? wsize * t.e + (long long)t.n0 * a.ldb : wsize * t.e + t.n0);
        const int mf = min(MF, (A.rows + 31) / 32);
        v16f c[MF];
#pragma unroll
        for (int i = 0; i < MF; i++)
#pragma unroll
            for (int j = 0; j < 16; j++) c[i][j] = 0.f;
        if (k > 0) A.load(0), B.load(0);
        for (int k0 = 0; k0 < k; k0 += BK) {
            __syncthreads();
            A.store(ta);
            B.store(tb);
            __syncthreads();
            if (k0 + BK < k) A.load(k0 + BK), B.load(k0 + BK);
#pragma unroll
            for (int s = 0; s < 2; s++) {
                const Frag fb = frag<BD, BN>(tb, wn, s, l);
#pragma unroll
                for (int i = 0; i < MF; i++)
                    if (i < mf) c[i] = mfma(fb, frag<AD, BM>(ta, 32 * i, s, l), c[i]);
            }
        }
        __syncthreads();
        const long long row0 = (KIND == DW ? (long long)t.e * a.m : t.lo) + t.m0;
#pragma unroll
        for (int i = 0; i < MF; i++)
            if (i < mf)
                Out<YTY, 1>::put((LE_LDS char *)smem + (threadIdx.x >> 6) * Out<YTY, 1>::BYTES, &c[i],
                                 (typename XT<YTY>::raw *)a.y + (row0 + 32 * i) * a.ldy + t.n0 + wn, a.ldy, A.rows - 32 * i, B.rows - wn);
    }
}

/* ---- rows of whole 16-byte chunks ----
 * 128 x BN tiles by four waves of 128 x BN / 4. Chunks go straight to LDS (lane l's 16 bytes to M0 + 16 l, so a wave's 64 land in a row; the
 * permutation is in which chunk a lane asks for), three steps in a ring: while one is multiplied, the next one's are about to land and those of the one
 * after it leave. One barrier a step: behind it a step's chunks are there for all waves, and the step before is read by all. Rows
 * beyond an expert's last are asked for as its last (their results are dropped), k beyond the depth as zeros. */

__device__ __attribute__((aligned(16))) const unsigned kZeros[4] = {0, 0, 0, 0};

/* In assembly, so that the compiler does not wait for it before every LDS read; step_ready below does. */
#pragma clang diagnostic push
#pragma clang diagnostic ignored "-Winline-asm"
__device__ __forceinline__ void chunk_to_lds(unsigned long long from, unsigned lds) {
    asm volatile("s_mov_b32 m0, %1\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %0, off" ::"v"(from), "s"(lds) : "memory", "m0");
}
#pragma clang diagnostic pop
/* All but this wave's last N chunks have landed, its reads of LDS are done, and so for the other waves. */
template <int N> __device__ __forceinline__ void step_ready() {
    asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" ::"n"(N) : "memory");
}

/* A wave's part of an operand's chunks: N of the 64 a time. */
template <bool DOWN, int R> struct Stream {
    static constexpr int N = R * 64 / 16 / 256;
    unsigned long long at[N]; /* address of this lane's chunk of the next step */
    int left[N];              /* depth that is left there */
    unsigned long long step;
    __device__ __forceinline__ void start(const void *base, long long ld, int rows, int depth) {
        step = DOWN ? (unsigned long long)ld * (BK * ES) : 64;
#pragma unroll
        for (int j = 0; j < N; j++) {
            const int id = threadIdx.x + 256 * j;
            int r, k;
            if constexpr (!DOWN) {
                r = id >> 2;
                k = ((id & 3) ^ ((r >> 2) & 3)) * EPC;
                r = min(r, rows - 1);
            } else {
                constexpr int C = R / EPC;
                k = id / C;
                const int sw = ES == 2 ? (k & 3) << 2 : ((k >> 2) & 1) << 3;
                r = min(((id % C) ^ (sw & (C - 1))) * EPC, rows - EPC);
            }
            left[j] = depth - k;
            at[j] = (unsigned long long)base + (DOWN ? k * ld + r : r * ld + k) * ES;
        }
    }
    /* The next step's chunks; whole: all of them lie within the depth. */
    __device__ __forceinline__ void load(unsigned lds, bool whole) {
        const unsigned wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
#pragma unroll
        for (int j = 0; j < N; j++) {
            chunk_to_lds(whole || left[j] > 0 ? at[j] : (unsigned long long)kZeros, lds + wave * 1024 + j * 4096);
            at[j] += step;
            left[j] -= BK;
        }
    }
};

template <Kind KIND, int YTY, int BN> __device__ __forceinline__ void pipe_body(const ExpertArgs &a) {
    constexpr int BM = 128, MF = 4, NF = BN / 128, STEP = (BM + BN) * 64, CHUNKS = (BM + BN) / 64;
    constexpr bool AD = KIND == DW, BD = KIND != Y;
    extern __shared__ __attribute__((aligned(16))) char ring[];
    LE_LDS char *const lds = (LE_LDS char *)ring;
    const int l = threadIdx.x & 63, wn = (threadIdx.x >> 6) * (BN / 4);
    for (long long b = blockIdx.x;; b += gridDim.x) {
        Tile t;
        if (!(KIND == DW ? find_weights<BM, BN>(a, tile_of(a, b), t) : find_rows<BM, BN>(a, tile_of(a, b), t))) return;
        const int m = KIND == DW ? a.m : t.cnt, depth = KIND == DW ? t.cnt : a.k, rows = m - t.m0, cols = a.n - t.n0;
        const long long wsize = (long long)a.n * a.k;
        const int steps = (depth + BK - 1) / BK;
        Stream<AD, BM> A;
        Stream<BD, BN> B;
        A.start((const T *)a.a + (KIND == DW ? t.lo * a.lda + t.m0 : (long long)(t.lo + t.m0) * a.lda), a.lda, rows, depth);
        B.start((const T *)a.b + (KIND == DW ? t.lo * a.ldb + t.n0 : wsize * t.e + (KIND == Y ? (long long)t.n0 * a.ldb : t.n0)), a.ldb, cols, depth);
        int slot = 0, to = 0, left = depth; /* places in the ring; depth that has not been asked for */
        auto ask = [&] {
            const unsigned at = (unsigned)(unsigned long long)lds + to;
            A.load(at, left >= BK);
            B.load(at + BM * 64, left >= BK);
            left -= BK;
            to = to == 2 * STEP ? 0 : to + STEP;
        };
        auto tile = [&](auto frags) {
            constexpr int F = decltype(frags)::value;
            v16f c[F][NF];
#pragma unroll
            for (int i = 0; i < F; i++)
#pragma unroll
                for (int n = 0; n < NF; n++)
#pragma unroll
                    for (int j = 0; j < 16; j++) c[i][n][j] = 0.f;
            /* two steps are asked for ahead, also behind the last (zeros): the count of chunks on their way is then always the same */
            ask();
            ask();
            for (int s = 0; s < steps; s++) {
                step_ready<CHUNKS>();
                ask();
                LE_LDS const char *ta = lds + slot, *tb = ta + BM * 64;
                slot = slot == 2 * STEP ? 0 : slot + STEP;
#pragma unroll
                for (int h = 0; h < 2; h++) {
                    Frag fb[NF];
#pragma unroll
                    for (int n = 0; n < NF; n++) fb[n] = frag<BD, BN>(tb, wn + 32 * n, h, l);
#pragma unroll
                    for (int i = 0; i < F; i++) {
                        const Frag fa = frag<AD, BM>(ta, 32 * i, h, l);
#pragma unroll
                        for (int n = 0; n < NF; n++) c[i][n] = mfma(fb[n], fa, c[i][n]);
                    }
                }
            }
            step_ready<0>(); /* the ring is free */
            const long long row0 = (KIND == DW ? (long long)t.e * a.m : t.lo) + t.m0;
#pragma unroll
            for (int i = 0; i < F; i++)
                Out<YTY, NF>::put(lds + (threadIdx.x >> 6) * Out<YTY, NF>::BYTES, c[i], (typename XT<YTY>::raw *)a.y + (row0 + 32 * i) * a.ldy + t.n0 + wn, a.ldy,
                                  rows - 32 * i, cols - wn);
            step_ready<0>();
        };
        switch (min(MF, (rows + 31) / 32)) {
        case 1: tile(Count<1>()); break;
        case 2: tile(Count<2>()); break;
        case 3: tile(Count<3>()); break;
        default: tile(Count<4>()); break;
        }
    }
}

}  // namespace

#define LE_EX_NAME2(WHAT, TY, TAIL) le_ex_##WHAT##_##TY##TAIL
#define LE_EX_NAME(WHAT, TY, TAIL) LE_EX_NAME2(WHAT, TY, TAIL)
#define LE_EX(WHAT, KIND, YTY)                                                                                                   \
    extern "C" __global__ void __launch_bounds__(256) LE_EX_NAME(WHAT, LE_EX_TY, _any)(ExpertArgs a) { any_body<KIND, YTY>(a); } \
    extern "C" __global__ void __launch_bounds__(256, 2) LE_EX_NAME(WHAT, LE_EX_TY, _n128)(ExpertArgs a) { pipe_body<KIND, YTY, 128>(a); } \
    extern "C" __global__ void __launch_bounds__(256, 2) LE_EX_NAME(WHAT, LE_EX_TY, _n256)(ExpertArgs a) { pipe_body<KIND, YTY, 256>(a); }
LE_EX(y, Y, TY)
LE_EX(dx, DX, TY)
LE_EX(dw, DW, TY)
#if LE_EX_TY != 0
LE_EX(dwf, DW, 0)
#endif
