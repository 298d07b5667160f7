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
constexpr int BK = 64 / ES;                  /* depth of a step of chunks that go straight to LDS */

typedef unsigned v4u __attribute__((ext_vector_type(4)));
typedef v4u __attribute__((aligned(ES))) v4u_any;
typedef float v4f __attribute__((ext_vector_type(4)));
typedef float v16f __attribute__((ext_vector_type(16)));
typedef short v4s __attribute__((ext_vector_type(4)));
typedef short v8s __attribute__((ext_vector_type(8)));
typedef _Float16 v8h __attribute__((ext_vector_type(8)));
typedef __bf16 v8b __attribute__((ext_vector_type(8)));

/* ---- tiles in LDS ---- */

/* W: bytes of k in a row of an `along` tile, 64, 128 or 256. Sixteen rows' chunks of one k fill the 64 banks once. */
template <bool DOWN, int R, int W> __device__ __forceinline__ int swizzle(int row_or_k) {
    if constexpr (!DOWN) return W == 64 ? (row_or_k >> 2) & 3 : W == 128 ? (row_or_k >> 1) & 7 : row_or_k & 15;
    else return (ES == 2 ? (row_or_k & 3) << 2 : ((row_or_k >> 2) & 1) << 3) & (R / EPC - 1);
}
template <bool DOWN, int R, int W = 64> __device__ __forceinline__ int lds_at(int row_or_k, int chunk) {
    return row_or_k * (DOWN ? R * ES : W) + ((chunk ^ swizzle<DOWN, R, W>(row_or_k)) << 4);
}

/* A lane's operand for a part of a step (fp32: of 8 values of k, else of 16): row row0 + lane % 32, k = (2 s + lane / 32) * EPC + 0 .. EPC - 1 */
union Frag {
    v4u u;
    v4f f;
    v8s s;
    struct {
        v4s lo, hi;
    } p;
};
template <bool DOWN, int R, int W = 64> __device__ __forceinline__ Frag frag(LE_LDS const char *tile, int row0, int s, int l) {
    Frag v;
    if constexpr (!DOWN) {
        v.u = *(LE_LDS const v4u *)(tile + lds_at<false, R, W>(row0 + (l & 31), 2 * s + (l >> 5)));
    } else if constexpr (ES == 4) {
        const int r = row0 + (l & 31), k = (2 * s + (l >> 5)) * 4;
#pragma unroll
        for (int j = 0; j < 4; j++) v.f[j] = *(LE_LDS const float *)(tile + lds_at<true, R, W>(k + j, r >> 2) + (r & 3) * 4);
    } else {
        /* 16 lanes read four k of 16 rows, 8 bytes each; lane i of them gets the four k of row i */
        const int i = l & 15, r = row0 + (l & 16) + (i & 3) * 4, k = (2 * s + (l >> 5)) * 8 + (i >> 2);
        typedef LE_LDS v4s *p4;
        v.p.lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((p4)(tile + lds_at<true, R, W>(k, r >> 3) + (r & 4) * 2));
        v.p.hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((p4)(tile + lds_at<true, R, W>(k + 4, r >> 3) + (r & 4) * 2));
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
/* An expert's rows, within the buffers whatever off holds (in memory or in LDS). */
template <class OFF> __device__ __forceinline__ void rows_of(const ExpertArgs &a, OFF off, int e, int &lo, int &cnt) {
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
template <int BM, int BN, class OFF> __device__ __forceinline__ bool find_rows(const ExpertArgs &a, OFF off, long long q, Tile &t) {
    const int l = threadIdx.x & 63, u = (int)(q / a.nt); /* row tiles before this one, over all experts */
    int before = 0;
    for (int e0 = 0; e0 < a.n_exp; e0 += 64) {
        int lo = 0, cnt = 0;
        if (e0 + l < a.n_exp) rows_of(a, off, e0 + l, lo, cnt);
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
template <int BM, int BN, class OFF> __device__ __forceinline__ bool find_weights(const ExpertArgs &a, OFF off, long long q, Tile &t) {
    const long long per = (long long)a.mt * a.nt;
    if (q >= per * a.n_exp * a.segs) return false;
    t.e = (int)(q / per); /* its sums' place: behind those of the parts before */
    const int seg = t.e / a.n_exp;
    rows_of(a, off, t.e - seg * a.n_exp, t.lo, t.cnt);
    if (a.segs > 1) {
        const int part = ((t.cnt - 1) / a.segs & ~31) + 32, before = (int)min((long long)seg * part, (long long)t.cnt); /* whole steps */
        t.lo += before;
        t.cnt = min(part, t.cnt - before);
    }
    place<BM, BN>(t, q - per * t.e, a.mt, a.nt);
    return true;
}

enum Kind { Y, DX, DW };
template <int N> struct Count { static constexpr int value = N; };
/* The tile that comes b-th for its block; false: behind the last. */
template <Kind KIND, int BM, int BN, class OFF> __device__ __forceinline__ bool find(const ExpertArgs &a, OFF off, long long b, Tile &t) {
    if constexpr (KIND == DW) return find_weights<BM, BN>(a, off, tile_of(a, b), t);
    else return find_rows<BM, BN>(a, off, tile_of(a, b), t);
}

/* ---- results ----
 * The operands go into the matrix instruction as (B, A): a lane then holds row l % 32 of the tile's 32 and 16 of 32 columns, four in a row. NF such
 * fragments side by side are rounded and change places through LDS of the wave's own, ROWS rows at a time, so that whole lines are written. */
template <int YTY, int NF, int ROWS = 32> struct Out {
    using U = typename XT<YTY>::raw;
    static constexpr int E = 16 / sizeof(U), LANES = 32 * NF / E, PITCH = 32 * NF * sizeof(U) + 16, BYTES = ROWS * PITCH;
    static constexpr int STORES = 32 * LANES / 64; /* instructions of a put */
    /* rows of them there are, at y, ld apart; cols of them there are, from this wave's first on. ALL: all 32 and 32 NF, in exactly STORES
     * instructions (in assembly, as they are counted on). */
    template <bool ALL = false> static __device__ __forceinline__ void put(LE_LDS char *mine, const v16f *c, void *y, long long ld, int rows, int cols) {
        typedef v4u __attribute__((aligned(4))) v4u_a4;
        typedef v4u __attribute__((aligned(2))) v4u_a2;
        const int l = threadIdx.x & 63, col = l % LANES * E;
#pragma unroll
        for (int r0 = 0; r0 < 32; r0 += ROWS) {
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront"); /* the reads of the rows before */
        __builtin_amdgcn_wave_barrier();
        if (ROWS == 32 || (l & 16) == r0) {
#pragma unroll
        for (int n = 0; n < NF; n++)
#pragma unroll
            for (int q = 0; q < 4; q++) { /* columns 8 q + 4 (l / 32) and on */
                LE_LDS char *p = mine + (l & (ROWS - 1)) * PITCH + (32 * n + 8 * q + 4 * (l >> 5)) * (int)sizeof(U);
                const float v0 = c[n][4 * q], v1 = c[n][4 * q + 1], v2 = c[n][4 * q + 2], v3 = c[n][4 * q + 3];
                if constexpr (sizeof(U) == 4) {
                    *(LE_LDS v4f *)p = v4f{v0, v1, v2, v3};
                } else {
                    typedef unsigned v2u __attribute__((ext_vector_type(2)));
                    *(LE_LDS v2u *)p = v2u{XT<YTY>::down(v0) | (unsigned)XT<YTY>::down(v1) << 16, XT<YTY>::down(v2) | (unsigned)XT<YTY>::down(v3) << 16};
                }
            }
        }
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        __builtin_amdgcn_wave_barrier();
#pragma unroll
        for (int i = 0; i < ROWS; i += 64 / LANES) {
            const int r = r0 + i + l / LANES;
            const v4u v = *(LE_LDS const v4u *)(mine + (r - r0) * PITCH + col * (int)sizeof(U));
            LE_GLOBAL U *to = (LE_GLOBAL U *)y + r * ld + col;
            if constexpr (ALL) {
                /* its registers may not be written in the two wait states behind it, and the compiler does not see a store here */
                asm volatile("global_store_dwordx4 %0, %1, off\n\ts_nop 1" ::"v"((unsigned long long)to), "v"(v) : "memory");
            } else if (r < rows) {
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
    }
};

/* This wave's reads and writes of LDS are done, and so for the other waves. */
__device__ __forceinline__ void meet() { asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory"); }

/* ---- any size, stride and alignment ----
 * BM x 128 tiles by four waves, chunks of 128 bytes of k a step through registers (16-byte loads at any address; a chunk that a row's end cuts is
 * loaded so that it ends there, and moved) into one half of LDS while the other is multiplied, the step behind that on its way
 * meanwhile. */

/* Chunks of R rows of an operand. */
template <bool DOWN, int R> struct Loader {
    static constexpr int BK = 128 / ES, N = R * 128 / 16 / 256, C = R / EPC; /* depth of a step, chunks a thread, chunks of R rows of `down` */
    struct Step {
        v4u v[N];
    };
    unsigned long long at[N], step; /* where a chunk of the next step begins, or is loaded from: `cut` values before that */
    int cut[N], have[N];            /* `down`; for rows shorter than a chunk: what there is of it */
    bool tiny;
    /* rows of them there are from base on, `before` before it in a row of `down`; depth values of k */
    __device__ __forceinline__ void start(const T *base, long long ld, int rows, int before, int depth) {
        step = DOWN ? (unsigned long long)ld * (BK * ES) : 128;
        tiny = (DOWN ? before + rows : depth) < EPC;
#pragma unroll
        for (int j = 0; j < N; j++) {
            const int id = threadIdx.x + 256 * j;
            if constexpr (!DOWN) {
                at[j] = (unsigned long long)(base + min(id >> 3, rows - 1) * ld + (id & 7) * EPC);
                cut[j] = 0;
            } else {
                const int r = min(id % C * EPC, rows - 1);
                have[j] = rows - r;
                cut[j] = tiny ? 0 : max(EPC - have[j], 0);
                at[j] = (unsigned long long)(base + id / C * ld + (r - cut[j]));
            }
        }
    }
    /* Of chunk j of a step, of whose depth `left` is left: how many values there are, 0 or less: none */
    static __device__ __forceinline__ int there(int j, int left) { return DOWN ? left - (int)(threadIdx.x + 256 * j) / C : left - (int)(threadIdx.x & 7) * EPC; }
    __device__ __forceinline__ void load(Step &s, int left) {
        if (left >= BK && !tiny) {
#pragma unroll
            for (int j = 0; j < N; j++) s.v[j] = *(const LE_GLOBAL v4u_any *)at[j];
        } else {
#pragma unroll
            for (int j = 0; j < N; j++) {
                const int n = there(j, left);
                const LE_GLOBAL T *p = (const LE_GLOBAL T *)at[j];
                s.v[j] = v4u{0, 0, 0, 0};
                if (n > 0) {
                    if (!tiny) {
                        s.v[j] = *(const LE_GLOBAL v4u_any *)(p - (DOWN ? 0 : max(EPC - n, 0)));
                    } else {
#pragma unroll
                        for (int e = 0; e < EPC - 1; e++)
                            if (e < (DOWN ? have[j] : n)) {
                                if constexpr (ES == 4) s.v[j][e] = ((const LE_GLOBAL unsigned *)p)[e];
                                else s.v[j][e >> 1] |= (unsigned)p[e] << (e & 1) * 16;
                            }
                    }
                }
            }
        }
#pragma unroll
        for (int j = 0; j < N; j++) at[j] += step;
    }
    /* What load() brought for a step with so much left. */
    __device__ __forceinline__ void store(const Step &s, LE_LDS char *tile, int left) const {
#pragma unroll
        for (int j = 0; j < N; j++) {
            const int id = threadIdx.x + 256 * j, early = DOWN ? cut[j] : tiny ? 0 : min(max(EPC - there(j, left), 0), EPC);
            v4u w = s.v[j];
            if ((DOWN || left < BK) && __any(early > 0)) { /* a chunk that was loaded early: its last values to the front, zeros behind them */
                const int bits = early * (8 * ES);
                unsigned long long lo = w[0] | (unsigned long long)w[1] << 32, hi = w[2] | (unsigned long long)w[3] << 32;
                const unsigned long long over = bits < 64 ? (hi << 1) << (63 - bits) : hi >> (bits & 63);
                lo = bits < 64 ? lo >> bits | over : bits < 128 ? over : 0;
                hi = bits < 64 ? hi >> bits : 0;
                w = v4u{(unsigned)lo, (unsigned)(lo >> 32), (unsigned)hi, (unsigned)(hi >> 32)};
            }
            *(LE_LDS v4u *)(tile + (!DOWN ? lds_at<false, R, 128>(id >> 3, id & 7) : lds_at<true, R, 128>(id / C, id % C))) = w;
        }
    }
};

template <Kind KIND, int YTY, int BM> __device__ __forceinline__ void any_body(const ExpertArgs &a) {
    constexpr int BN = 128, WM = BM == 128 ? 2 : 1, WN = 4 / WM, MF = BM / 32 / WM, NF = BN / 32 / WN, HALF = (BM + BN) * 128, BK = 128 / ES;
    constexpr bool AD = KIND == DW, BD = KIND != Y;
    using O = Out<YTY, NF, 32>;
    static_assert(4 * O::BYTES <= 2 * HALF, "results");
    __shared__ __attribute__((aligned(16))) char smem[2 * HALF];
    LE_LDS char *const lds = (LE_LDS char *)smem;
    const int l = threadIdx.x & 63, wave = threadIdx.x >> 6, wm = wave / WN, wn = wave % WN * (BN / WN);
    for (long long b = blockIdx.x;; b += gridDim.x) {
        Tile t;
        if (!find<KIND, BM, BN>(a, (const LE_GLOBAL int *)a.off, b, t)) return;
        const int m = KIND == DW ? a.m : t.cnt, k = KIND == DW ? t.cnt : a.k, rows = m - t.m0, cols = a.n - t.n0;
        using LA = Loader<AD, BM>;
        using LB = Loader<BD, BN>;
        LA A;
        LB B;
        A.start((const T *)a.a + (KIND == DW ? t.lo * a.lda + t.m0 : (long long)(t.lo + t.m0) * a.lda), a.lda, rows, t.m0, k);
        B.start((const T *)a.b + (KIND == DW ? t.lo * a.ldb + t.n0 : (long long)a.n * a.k * t.e + (KIND == Y ? (long long)t.n0 * a.ldb : t.n0)), a.ldb, cols, t.n0, k);
        const int f = max(0, min(MF, ((rows + 31) / 32 - wm + WM - 1) / WM));
        v16f c[MF][NF];
#pragma unroll
        for (int i = 0; i < MF; i++)
#pragma unroll
            for (int n = 0; n < NF; n++)
#pragma unroll
                for (int j = 0; j < 16; j++) c[i][n][j] = 0.f;
        typename LA::Step sa;
        typename LB::Step sb;
        A.load(sa, k), B.load(sb, k);
        A.store(sa, lds, k), B.store(sb, lds + BM * 128, k);
        A.load(sa, k - BK), B.load(sb, k - BK);
        for (int left = k, half = 0; left > 0;) {
            meet();
            LE_LDS const char *ta = lds + half, *tb = ta + BM * 128;
#pragma unroll
            for (int p = 0; p < 4; p++) {
                Frag fb[NF];
#pragma unroll
                for (int n = 0; n < NF; n++) fb[n] = frag<BD, BN, 128>(tb, wn + 32 * n, p, l);
#pragma unroll
                for (int i = 0; i < MF; i++)
                    if (i < f) {
                        const Frag fa = frag<AD, BM, 128>(ta, 32 * (WM * i + wm), p, l);
#pragma unroll
                        for (int n = 0; n < NF; n++) c[i][n] = mfma(fb[n], fa, c[i][n]);
                    }
            }
            half ^= HALF;
            left -= BK;
            if (left > 0) { /* two steps ahead gained nothing (dx of 1806 rows, 60 experts of 515 x 1001 fp32, 61 / 66 us) */
                A.store(sa, lds + half, left), B.store(sb, lds + half + BM * 128, left);
                A.load(sa, left - BK), B.load(sb, left - BK);
            }
        }
        meet();
        const long long row0 = (KIND == DW ? (long long)t.e * a.m : t.lo) + t.m0 + 32 * wm;
#pragma unroll
        for (int i = 0; i < MF; i++)
            if (i < f)
                O::put(lds + wave * O::BYTES, c[i], (typename XT<YTY>::raw *)a.y + (row0 + 32 * WM * i) * a.ldy + t.n0 + wn, a.ldy, rows - 32 * (WM * i + wm), cols - wn);
        meet();
    }
}

/* ---- rows of whole 16-byte chunks ----
 * BM x BN tiles by four waves of BM x BN / 4. Chunks go straight to LDS (lane l's 16 bytes to M0 + 16 l, so a wave's 64 land in a row; the
 * permutation is in which chunk a lane asks for), RING steps in a ring: while one is multiplied, the others are on their way. One barrier
 * a step: behind it a step's chunks are there for all waves, and the step before is read by all. Rows
 * beyond an expert's last are asked for as its last (their results are dropped), k beyond the depth as zeros.
 * 128 experts of 1536 x 2048 bf16, 32768 rows (206 GFLOP, 1.0 GB): y 293 to 325 us, dx 289 to 300; a copy of those bytes would take 200, the products at the
 * clock that they leave 150. What comes from beyond the L2 (1.3 GB, as an expert's second tile of rows finds its weights gone) moves at
 * what the fabric gives, 6 TB/s, for y less: its operands are read 64 bytes of a row at a time, which alone runs at 4.4 TB/s. Steps of 128
 * bytes leave LDS for one in flight: 332. */

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

/* A wave's part of an operand's chunks, NT threads in all. */
template <bool DOWN, int R, int NT> struct Stream {
    static constexpr int N = R * 4 / NT, C = R / EPC; /* chunks a thread; chunks of R rows of `down` */
    unsigned long long at[N] = {}; /* address of this lane's chunk of the next step */
    unsigned long long step = 0;
    /* k of chunk 0 in its step; also of a stream that is never started, which loads zeros (left 0) */
    const int k = DOWN ? (int)threadIdx.x / C : ((threadIdx.x & 3) ^ ((threadIdx.x >> 4) & 3)) * EPC;
    __device__ __forceinline__ void start(const void *base, long long ld, int rows) {
        step = DOWN ? (unsigned long long)ld * (BK * ES) : 64;
#pragma unroll
        for (int j = 0; j < N; j++) {
            const int id = threadIdx.x + NT * j;
            if constexpr (!DOWN) {
                at[j] = (unsigned long long)base + (min(id >> 2, rows - 1) * ld + k) * ES;
            } else {
                const int kj = id / C, sw = ES == 2 ? (kj & 3) << 2 : ((kj >> 2) & 1) << 3;
                at[j] = (unsigned long long)base + (kj * ld + min(((id % C) ^ (sw & (C - 1))) * EPC, rows - EPC)) * ES;
            }
        }
    }
    __device__ __forceinline__ void skip(int steps) {
#pragma unroll
        for (int j = 0; j < N; j++) at[j] += (long long)steps * (long long)step;
    }
    /* The next step's chunks; left: depth from its start on, zeros where that ends. */
    __device__ __forceinline__ void load(unsigned lds, int left) {
        const unsigned wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
        if (left >= BK) {
#pragma unroll
            for (int j = 0; j < N; j++) {
                chunk_to_lds(at[j], lds + wave * 1024 + j * NT * 16);
                at[j] += step;
            }
        } else {
#pragma unroll
            for (int j = 0; j < N; j++) {
                chunk_to_lds(k + (DOWN ? j * (NT / C) : 0) < left ? at[j] : (unsigned long long)kZeros, lds + wave * 1024 + j * NT * 16);
                at[j] += step;
            }
        }
    }
};

template <Kind KIND, int YTY, int BM, int BN, int RING> __device__ __forceinline__ void pipe_body(const ExpertArgs &a) {
    constexpr int MF = BM / 32, NF = BN / 128, STEP = (BM + BN) * 64, CHUNKS = (BM + BN) / 64;
    constexpr bool AD = KIND == DW, BD = KIND != Y;
    extern __shared__ __attribute__((aligned(16))) char ring[];
    LE_LDS char *const lds = (LE_LDS char *)ring;
    const int l = threadIdx.x & 63, wn = (threadIdx.x >> 6) * (BN / 4);
    for (long long b = blockIdx.x;; b += gridDim.x) {
        Tile t;
        if (!find<KIND, BM, BN>(a, (const LE_GLOBAL int *)a.off, b, t)) return;
        const int m = KIND == DW ? a.m : t.cnt, depth = KIND == DW ? t.cnt : a.k, rows = m - t.m0, cols = a.n - t.n0;
        const long long wsize = (long long)a.n * a.k;
        const int steps = (depth + BK - 1) / BK;
        Stream<AD, BM, 256> A;
        Stream<BD, BN, 256> B;
        A.start((const T *)a.a + (KIND == DW ? t.lo * a.lda + t.m0 : (long long)(t.lo + t.m0) * a.lda), a.lda, rows);
        B.start((const T *)a.b + (KIND == DW ? t.lo * a.ldb + t.n0 : wsize * t.e + (KIND == Y ? (long long)t.n0 * a.ldb : t.n0)), a.ldb, cols);
        /* Rows of W and x lie a power of two apart as a rule, so that every tile's first steps would ask the same channels: experts begin at steps of
         * their own (y of 1024 rows of 128 experts of 1536 x 2048 bf16 172 / 136 us, 8192 rows 208 / 190, 32768 321 / 325). */
        int step = KIND == Y ? t.e * 5 % steps : 0, asked = 0;
        A.skip(step);
        B.skip(step);
        int slot = 0, to = 0; /* places in the ring */
        auto ask = [&] {
            const unsigned at = (unsigned)(unsigned long long)lds + to;
            const int left = asked < steps ? depth - step * BK : 0;
            A.load(at, left);
            B.load(at + BM * 64, left);
            asked++;
            step++;
            if (KIND == Y && step == steps) {
                step = 0;
                A.skip(-steps);
                B.skip(-steps);
            }
            to = to == (RING - 1) * STEP ? 0 : to + STEP;
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
            /* RING - 1 steps are asked for ahead, also behind the last (zeros): the count of chunks on their way is then always the same */
#pragma unroll
            for (int i = 0; i < RING - 1; i++) ask();
            for (int s = 0; s < steps; s++) {
                step_ready<(RING - 2) * CHUNKS>();
                ask();
                LE_LDS const char *ta = lds + slot, *tb = ta + BM * 64;
                slot = slot == (RING - 1) * STEP ? 0 : slot + STEP;
                Frag fa[2][F], fb[2][NF];
#pragma unroll
                for (int h = 0; h < 2; h++) {
#pragma unroll
                    for (int n = 0; n < NF; n++) fb[h][n] = frag<BD, BN>(tb, wn + 32 * n, h, l);
#pragma unroll
                    for (int i = 0; i < F; i++) fa[h][i] = frag<AD, BM>(ta, 32 * i, h, l);
                }
#pragma unroll
                for (int h = 0; h < 2; h++)
#pragma unroll
                    for (int i = 0; i < F; i++)
#pragma unroll
                        for (int n = 0; n < NF; n++) c[i][n] = mfma(fb[h][n], fa[h][i], c[i][n]);
            }
            step_ready<0>(); /* the ring is free */
            const long long row0 = (KIND == DW ? (long long)t.e * a.m : t.lo) + t.m0;
#pragma unroll
            for (int i = 0; i < F; i++)
                Out<YTY, NF>::put(lds + (threadIdx.x >> 6) * Out<YTY, NF>::BYTES, c[i], (typename XT<YTY>::raw *)a.y + (row0 + 32 * i) * a.ldy + t.n0 + wn, a.ldy,
                                  rows - 32 * i, cols - wn);
            step_ready<0>();
        };
        const int f = min(MF, (rows + 31) / 32);
        if (f == 1) tile(Count<1>());
        else if (MF == 2 || f == 2) tile(Count<2>());
        else if (f == 3) tile(Count<(MF > 2 ? 3 : 2)>());
        else tile(Count<MF>());
    }
}

/* ---- few rows an expert ----
 * y of at most 32 rows of an expert by 32 outputs, or a.strip times 32 one after the other, by one wave: nothing is shared, so there is no barrier,
 * and a CU's four waves stream weights on their own. 256 bytes of a row of W at a time, since what comes from beyond the L2
 * arrives the faster the longer its pieces are (64 bytes of each of many rows 4.4 TB/s, 128 5.3, 256 6.0); tiles begin at steps of
 * their own, since rows lie a power of two apart as a rule and waves in the same place would ask the same channels (64 rows of 128 experts
 * of 1536 x 2048 bf16 66 / 60 us). Of x only the rows that there are, in fours, so that the fewer they are, the more steps are on their way: 8 + X
 * kB each. Where there are few tiles, a block's waves take steps in turn, and their sums meet in LDS. */
constexpr int FEW_LDS = 40960; /* a wave's: the ring, then its results */
template <int X> __device__ __forceinline__ void few_tile(const ExpertArgs &a, const Tile &t, LE_LDS char *lds, int wave, int nw) {
    using O = Out<TY, 1, 16>;
    constexpr int BKF = 256 / ES, STEP = (8 + X) * 1024, RING = (FEW_LDS - O::BYTES) / STEP;
    const int l = threadIdx.x & 63, rows = t.cnt - t.m0, steps = (a.k + BKF - 1) / BKF, tiles = min(a.strip, (a.n - t.n0 + 31) / 32);
    LE_LDS char *const mine = lds + wave * FEW_LDS;
    auto row_of = [&](int j) { return 4 * j + (l >> 4); }; /* chunk j of x or W: four rows an instruction */
    auto k_of = [&](int j) { return ((l & 15) ^ (row_of(j) & 15)) * EPC; };
    const T *const w = (const T *)a.b + (long long)a.n * a.k * t.e;
    unsigned long long xat[X], wat[8]; /* of this lane's chunks of a tile's step 0 */
#pragma unroll
    for (int j = 0; j < X; j++) xat[j] = (unsigned long long)((const T *)a.a + (long long)(t.lo + t.m0 + min(row_of(j), rows - 1)) * a.lda + k_of(j));
    auto point = [&](int q) {
#pragma unroll
        for (int j = 0; j < 8; j++) wat[j] = (unsigned long long)(w + (long long)min(t.n0 + 32 * q + row_of(j), a.n - 1) * a.ldb + k_of(j));
    };
    auto begin = [&](int q) { return (t.n0 / 32 + q) % steps; };
    int to = 0, asked = 0, next = wave, first = begin(0); /* tile and step to ask for */
    point(0);
    auto ask = [&] {
        if (next >= steps && asked < tiles) {
            next = wave;
            if (++asked < tiles) point(asked), first = begin(asked);
        }
        const unsigned base = (unsigned)(unsigned long long)mine + to;
        const int step = next + first >= steps ? next + first - steps : next + first, left = asked < tiles ? a.k - step * BKF : 0; /* 0: zeros */
#pragma unroll
        for (int j = 0; j < X; j++) chunk_to_lds(left >= BKF || k_of(j) < left ? xat[j] + step * 256LL : (unsigned long long)kZeros, base + j * 1024);
#pragma unroll
        for (int j = 0; j < 8; j++) chunk_to_lds(left >= BKF || k_of(j) < left ? wat[j] + step * 256LL : (unsigned long long)kZeros, base + (X + j) * 1024);
        next += nw;
        to = to == (RING - 1) * STEP ? 0 : to + STEP;
    };
#pragma unroll
    for (int i = 0; i < RING - 1; i++) ask();
    int slot = 0;
    for (int q = 0; q < tiles; q++) {
        v16f c[2];
#pragma unroll
        for (int j = 0; j < 16; j++) c[0][j] = 0.f, c[1][j] = 0.f;
        for (int s = wave; s < steps; s += nw) {
            asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)" ::"n"((RING - 2) * (8 + X)) : "memory");
            ask();
            LE_LDS const char *tx = mine + slot, *tw = tx + X * 1024;
            slot = slot == (RING - 1) * STEP ? 0 : slot + STEP;
#pragma unroll
            for (int h = 0; h < 8; h++) { /* rows of x that are not there: the others once more */
                const Frag fx = frag<false, 32, 256>(tx, 0, h, X == 8 ? l : (l & 32) | (l & (4 * X - 1))), fw = frag<false, 32, 256>(tw, 0, h, l);
                c[h & 1] = mfma(fw, fx, c[h & 1]);
            }
        }
#pragma unroll
        for (int j = 0; j < 16; j++) c[0][j] += c[1][j];
        if (nw > 1) { /* one tile here; the waves' sums, in their order */
            asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory"); /* the ring is free */
            if (wave)
#pragma unroll
                for (int j = 0; j < 4; j++) *(LE_LDS v4f *)(mine + (j * 64 + l) * 16) = v4f{c[0][4 * j], c[0][4 * j + 1], c[0][4 * j + 2], c[0][4 * j + 3]};
            meet();
            if (!wave)
                for (int o = 1; o < nw; o++)
#pragma unroll
                    for (int j = 0; j < 4; j++) {
                        const v4f v = *(LE_LDS const v4f *)(lds + o * FEW_LDS + (j * 64 + l) * 16);
#pragma unroll
                        for (int e = 0; e < 4; e++) c[0][4 * j + e] += v[e];
                    }
        }
        if (!wave)
            O::put(mine + RING * STEP, c, (T *)a.y + (long long)(t.lo + t.m0) * a.ldy + t.n0 + 32 * q, a.ldy, rows, a.n - t.n0 - 32 * q);
    }
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory"); /* nothing may land in LDS that is another tile's */
}
__device__ __forceinline__ void few_body(const ExpertArgs &a) {
    extern __shared__ __attribute__((aligned(16))) char ring[];
    LE_LDS char *const lds = (LE_LDS char *)ring;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), nw = blockDim.x >> 6;
    for (long long b = blockIdx.x;; b += gridDim.x) {
        Tile t;
        if (!find<Y, 32, 1>(a, (const LE_GLOBAL int *)a.off, b, t)) return;
        t.n0 *= 32 * a.strip;
        const int rows = t.cnt - t.m0;
        if (rows <= 4) few_tile<1>(a, t, lds, wave, nw);
        else if (rows <= 8) few_tile<2>(a, t, lds, wave, nw);
        else if (rows <= 16) few_tile<4>(a, t, lds, wave, nw);
        else few_tile<8>(a, t, lds, wave, nw);
        meet(); /* the reads of LDS */
    }
}

/* ---- weights' gradient ----
 * An expert's rows make a short depth and a large result: 256 x 256 tiles by eight waves (2 x 4; a wave has every other 32 rows and 64 columns),
 * a block a CU, which takes tile after tile. What goes to LDS runs AHEAD steps ahead of what is multiplied, also from one tile into the
 * next, so that nothing waits for a tile's first chunks and the results leave meanwhile. off lies in LDS, since a wait for a load from
 * memory would be one for the chunks as well. 128 experts of 1536 x 2048 bf16, 32768 rows: 350 us (while the first steps waited for the stores
 * before them 357), in the tiles above 404; 8168 rows of 2048 x 768 fp16 115 / 129. Without its stores it takes 262, without the
 * matrix instructions 307, without both 144: loads and stores (1.16 GB, at a copy's rate 223) overlap in part only, since a tile's stores are
 * waited for AHEAD steps later, and LDS holds no longer ring. (The other two products gained nothing from such tiles before y's steps were
 * staggered; not measured since.) */
template <Kind KIND, int YTY, int RING> __device__ __forceinline__ void wide_body(const ExpertArgs &a) {
    constexpr int BM = 256, BN = 256, NT = 512, STEP = (BM + BN) * 64, CHUNKS = (BM + BN) * 4 / NT, AHEAD = RING - 1;
    constexpr bool AD = KIND == DW, BD = KIND != Y;
    extern __shared__ __attribute__((aligned(16))) char ring[]; /* the ring, the waves' results, off */
    LE_LDS char *const lds = (LE_LDS char *)ring;
    using O = Out<YTY, 2, 16>;
    LE_LDS int *const off = (LE_LDS int *)(lds + RING * STEP + 8 * O::BYTES);
    const int l = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), wm = wave >> 2, wn = (wave & 3) * 64;
    for (int i = threadIdx.x; i <= a.n_exp; i += NT) off[i] = ((const LE_GLOBAL int *)a.off)[i];
    __syncthreads();
    Stream<AD, BM, NT> A;
    Stream<BD, BN, NT> B;
    long long next = blockIdx.x; /* tile to ask for after this one */
    int to = 0, left = 0;        /* place in the ring; depth of the tile that is left to be asked for */
    bool more = true;
    auto ask = [&] {
        while (left <= 0 && more) { /* an expert without rows has tiles of its weights, but nothing to ask for */
            Tile t;
            more = find<KIND, BM, BN>(a, off, next, t);
            next += gridDim.x;
            if (more) {
                A.start((const T *)a.a + (KIND == DW ? t.lo * a.lda + t.m0 : (long long)(t.lo + t.m0) * a.lda), a.lda, (KIND == DW ? a.m : t.cnt) - t.m0);
                B.start((const T *)a.b + (KIND == DW ? t.lo * a.ldb + t.n0 : (long long)a.n * a.k * t.e + (KIND == Y ? (long long)t.n0 * a.ldb : t.n0)), a.ldb, a.n - t.n0);
                left = KIND == DW ? t.cnt : a.k;
            }
        }
        const unsigned at = (unsigned)(unsigned long long)lds + to; /* zeros behind the last tile: the count of chunks on their way is always the same */
        A.load(at, left);
        B.load(at + BM * 64, left);
        left -= BK;
        to = to == (RING - 1) * STEP ? 0 : to + STEP;
    };
#pragma unroll
    for (int i = 0; i < AHEAD; i++) ask();
    int slot = 0, late = 0; /* steps to come that were asked for before a tile's results left */
    for (long long b = blockIdx.x;; b += gridDim.x) {
        Tile t;
        if (!find<KIND, BM, BN>(a, off, b, t)) break;
        const int m = KIND == DW ? a.m : t.cnt, depth = KIND == DW ? t.cnt : a.k, rows = m - t.m0, cols = a.n - t.n0;
        const int f = max(0, min(4, ((rows + 31) / 32 - wm + 1) / 2)); /* of this wave's four times 32 rows those that there are */
        v16f c[4][2];
#pragma unroll
        for (int i = 0; i < 4; i++)
#pragma unroll
            for (int n = 0; n < 2; n++)
#pragma unroll
                for (int j = 0; j < 16; j++) c[i][n][j] = 0.f;
        auto steps = [&](auto full) {
            for (int s = 0; s < depth; s += BK) {
                if (late > 0) step_ready<(AHEAD - 1) * CHUNKS + 4 * O::STORES>(), late--;
                else step_ready<(AHEAD - 1) * CHUNKS>();
                ask();
                LE_LDS const char *ta = lds + slot, *tb = ta + BM * 64;
                slot = slot == (RING - 1) * STEP ? 0 : slot + STEP;
                Frag fa[2][4], fb[2][2];
#pragma unroll
                for (int h = 0; h < 2; h++) {
#pragma unroll
                    for (int n = 0; n < 2; n++) fb[h][n] = frag<BD, BN>(tb, wn + 32 * n, h, l);
#pragma unroll
                    for (int i = 0; i < 4; i++) fa[h][i] = frag<AD, BM>(ta, 64 * i + 32 * wm, h, l);
                }
                __builtin_amdgcn_sched_barrier(0); /* all reads ahead of the products */
#pragma unroll
                for (int h = 0; h < 2; h++)
#pragma unroll
                    for (int i = 0; i < 4; i++)
                        if (decltype(full)::value || i < f) {
#pragma unroll
                            for (int n = 0; n < 2; n++) c[i][n] = mfma(fb[h][n], fa[h][i], c[i][n]);
                        }
            }
        };
        if (f == 4) steps(Count<1>());
        else steps(Count<0>());
        const long long row0 = (KIND == DW ? (long long)t.e * a.m : t.lo) + t.m0 + 32 * wm;
        typename XT<YTY>::raw *const y = (typename XT<YTY>::raw *)a.y + row0 * a.ldy + t.n0 + wn;
        LE_LDS char *const mine = lds + RING * STEP + wave * O::BYTES;
        if (rows >= BM && cols >= BN) { /* the AHEAD steps that come next do not wait for these stores */
#pragma unroll
            for (int i = 0; i < 4; i++) O::template put<true>(mine, c[i], y + 64 * i * a.ldy, a.ldy, 32, 64);
            late = AHEAD;
        } else {
#pragma unroll
            for (int i = 0; i < 4; i++)
                if (i < f) O::put(mine, c[i], y + 64 * i * a.ldy, a.ldy, rows - 64 * i - 32 * wm, cols - wn);
            late = 0;
        }
    }
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory"); /* nothing may land in LDS that is no longer this block's */
}

/* ---- the sums of a weights' gradient's parts, in their order ---- */
template <int YTY> __device__ __forceinline__ void sum_body(const float *parts, void *y, int n, int segs) {
    const int i = blockIdx.x * 256 + threadIdx.x;
    if (i >= n) return;
    float v = 0.f;
#pragma unroll 8
    for (int s = 0; s < segs; s++) v += ((const LE_GLOBAL float *)parts)[(long long)s * n + i];
    ((LE_GLOBAL typename XT<YTY>::raw *)y)[i] = XT<YTY>::down(v);
}

}  // namespace

#define LE_EX_NAME2(WHAT, TY, TAIL) le_ex_##WHAT##_##TY##TAIL
#define LE_EX_NAME(WHAT, TY, TAIL) LE_EX_NAME2(WHAT, TY, TAIL)
#define LE_EX(WHAT, KIND, YTY)                                                                                                   \
    extern "C" __global__ void __launch_bounds__(256) LE_EX_NAME(WHAT, LE_EX_TY, _any32)(ExpertArgs a) { any_body<KIND, YTY, 32>(a); }   \
    extern "C" __global__ void __launch_bounds__(256, 2) LE_EX_NAME(WHAT, LE_EX_TY, _any128)(ExpertArgs a) { any_body<KIND, YTY, 128>(a); } \
    extern "C" __global__ void __launch_bounds__(256, 2) LE_EX_NAME(WHAT, LE_EX_TY, _m128_n128)(ExpertArgs a) { pipe_body<KIND, YTY, 128, 128, 3>(a); }
#define LE_EX_ROWS(WHAT, KIND) \
    extern "C" __global__ void __launch_bounds__(256, 2) LE_EX_NAME(WHAT, LE_EX_TY, _m128_n256)(ExpertArgs a) { pipe_body<KIND, TY, 128, 256, 3>(a); }
#define LE_EX_DW(WHAT, YTY)                                                                                                                 \
    LE_EX(WHAT, DW, YTY)                                                                                                                    \
    extern "C" __global__ void __launch_bounds__(512) LE_EX_NAME(WHAT, LE_EX_TY, _m256_n256)(ExpertArgs a) { wide_body<DW, YTY, YTY == 0 ? 3 : 4>(a); }                             \
    extern "C" __global__ void __launch_bounds__(256) LE_EX_NAME(WHAT, LE_EX_TY, _sum)(const float *parts, void *y, int n, int segs) { sum_body<YTY>(parts, y, n, segs); }
LE_EX(y, Y, TY)
LE_EX(dx, DX, TY)
extern "C" __global__ void __launch_bounds__(256, 1) LE_EX_NAME(y, LE_EX_TY, _few)(ExpertArgs a) { few_body(a); }
LE_EX_DW(dw, TY)
#if LE_EX_TY != 0
LE_EX_ROWS(y, Y)
LE_EX_ROWS(dx, DX)
LE_EX_DW(dwf, 0)
#endif
