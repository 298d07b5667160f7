/* Matrix-vector products with 4-bit codes and group scales (le_matvec_g4, include/le_qmm.h):
 *     y[r] = sum over groups g of scale[r][g] * sum over the group's c of (code[r][c] - zero[r][g]) * a[c]. */
#include <hip/hip_runtime.h>

#include "le_f32_types.h"
#include "le_g4_args.h"

/* ---- one to four virtual rows: the matrix cores, activations in registers ----
 *
 * With q = 16 + code, a bf16 whose low mantissa bits are the code's (one AND-OR on the shifted word makes two of them),
 *     y[r] = sum over scale blocks b of scale * (sum q a - (16 + zero) * sum a),
 * so the codes go to the matrix cores as they lie, and scale and zero point are applied to sums of 32 to 128 columns. An
 * activation enters as P = 1 to 3 bf16 pieces that add up to it (fp32: 24 bits in three of eight), so every product is exact.
 *
 * v_mfma_f32_16x16x32_bf16 with activations as A and weights as B. A few tokens use a few of A's 16 rows, so here the rows are
 * four K parts of 128 columns (kappa) times four virtual rows i = (token, piece), and B's columns are four weight rows (rho) times
 * the same four K parts. Of the 16 x 16 results only those count whose row and column have one kappa: MFMAs to spare buy
 * loads of 256 contiguous bytes a weight row instead of 64, and activations that stay in registers: a
 * wave keeps a slice of 512 columns (lane (m, g) the octets of row m = 4 kappa + i that MFMA j takes from lane group g).
 * Lane (n, g) of B takes kappa = (n + u) & 3 in step u of four; the result that counts then lies, in register i, in the lanes with
 * g = kappa, which are different lanes in each step. So after four steps, 16 weight rows, every lane has exactly one, picked by a
 * select, and scale, zero point and sum are applied once for all of them: lane (n, g) holds row 4 u + (n >> 2), u = (g - n) & 3,
 * and K part g.
 * The sums of a over the scale blocks come from the same MFMAs with B = 1, and so lie where they are needed.
 *
 * Scale blocks of 64 and 32 columns: the words of a lane's 16 bytes are exchanged between the lane groups (v_permlane32_swap,
 * v_permlane16_swap) until each MFMA's 32 columns lie in one block. Every word gives its eight columns in the order 0, 4, 1, 5, 2, 6,
 * 3, 7, and the activations are packed to match.
 *
 * The waves of a block split K, in passes where they are fewer than the slices, and go over the same row groups, each at its own
 * pace: partial results are kept in LDS, every lane's in a place of its own, and meet after one barrier, added in wave order.
 * Codes of the next two items are on their way while one is multiplied; loads of items that do not exist and of rows past the end
 * are cut off by the buffer's size and fetch nothing.
 *
 * One token, weights from HBM (graph replays over 700 MB of them; in brackets a streaming read of as many bytes): 28672 x 4096 bf16, groups of
 * 128, 62 MB 13.1 us (11.8), 14336 x 4096 fp32 31 MB 8.2 (6.9), groups of 32 37 MB 9.4, 4096 x 4096 4.7 (3.5), 1024 x 2048 3.15 (2.7), 4096 x 14336
 * SwiGLU fp32, groups of 64, 33 MB 13.0 (7.3): there each of 256 blocks reads all of x, forms SwiGLU and goes over K twice for its
 * 16 rows. What the types and groups choose is compiled in: as branches on arguments it cost 14336 x 4096 in groups of 32 5.6 us. */
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef float f32x4 __attribute__((ext_vector_type(4)));

static __device__ __forceinline__ unsigned bits(float v) { return __builtin_bit_cast(unsigned, v); }
static __device__ __forceinline__ float flt(unsigned v) { return __builtin_bit_cast(float, v); }
static __device__ __forceinline__ float cut16(float v) { return flt(bits(v) & 0xFFFF0000u); }
/* low half: the upper 16 bits of lo; high half: those of hi */
static __device__ __forceinline__ unsigned pack_hi16(float lo, float hi) { return __builtin_amdgcn_perm(bits(hi), bits(lo), 0x07060302u); }
/* Eight values, cut to bf16, in a word's order of columns. */
static __device__ __forceinline__ uint4 pack_octet(const float (&f)[8]) {
    return make_uint4(pack_hi16(f[0], f[4]), pack_hi16(f[1], f[5]), pack_hi16(f[2], f[6]), pack_hi16(f[3], f[7]));
}
/* The same, rounded to nearest. */
static __device__ __forceinline__ uint4 pack_octet_near(const float (&f)[8]) {
    auto two = [&](int k) { return __builtin_bit_cast(unsigned, (bf16x2){(__bf16)f[k], (__bf16)f[k + 4]}); };
    return make_uint4(two(0), two(1), two(2), two(3));
}
/* First column, of a part of 128, of the octet that MFMA j takes from lane group g. */
template <int SUB> static __device__ __forceinline__ int octet_col(int j, int g) {
    if (SUB == 128) return 32 * g + 8 * j;
    if (SUB == 64) return 32 * (2 * (j >> 1) + (g & 1)) + 8 * ((j & 1) + 2 * (g >> 1));
    return 32 * j + 8 * g;
}
/* 16 bytes of codes with the words exchanged so that word j holds MFMA j's columns. */
template <int SUB> static __device__ __forceinline__ void spread(uint4 &q) {
    if (SUB <= 64) {
        auto a = __builtin_amdgcn_permlane32_swap(q.x, q.z, false, false);
        auto b = __builtin_amdgcn_permlane32_swap(q.y, q.w, false, false);
        q = make_uint4(a[0], b[0], a[1], b[1]);
    }
    if (SUB == 32) {
        auto a = __builtin_amdgcn_permlane16_swap(q.x, q.y, false, false);
        auto b = __builtin_amdgcn_permlane16_swap(q.z, q.w, false, false);
        q = make_uint4(a[0], a[1], b[0], b[1]);
    }
}
/* Eight codes as bf16 16 + code. k: the mask 0x00780078 in a vector register, so that AND and OR are one instruction (which takes one
 * constant). */
static __device__ __forceinline__ bf16x8 unpack(unsigned q, unsigned k) {
    const unsigned o = 0x41804180u;
    return __builtin_bit_cast(bf16x8, make_uint4(((q << 3) & k) | o, ((q >> 1) & k) | o, ((q >> 5) & k) | o, ((q >> 9) & k) | o));
}
static __device__ __forceinline__ f32x4 mfma(const uint4 &a, const bf16x8 &b, const f32x4 &c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a), b, c, 0, 0, 0);
}
/* silu(g) * u = g u / (1 + 2^t), t = -g log2 e held as t0 + lo; the exponential and the reciprocal are the hardware's (1 ulp each), and with
 * the roundings of 1 + e and of the two products the result is within 2^-21 of its value. Below -126 there is no lo to add, and t0, which g of
 * 2^127 and more make infinite, gives none.
 * FAR: t0 beyond 126 too, where 1 + 2^t is 2^t to fp32 and its reciprocal may be below fp32's normal values though the product with a large
 * u is not: g 2^-t u, with 2^-t as 2^(n - t) in (1/2, 1], which cannot overflow g, and half of 2^-n to each factor. From n = 512 on that
 * is 0 for all finite g and u (2^128 2^-256 each); g of -infinity stays infinite, or NaN. */
constexpr float kLog2e = 1.44269502f, kLn2 = 0.693147181f;
template <bool FAR> static __device__ __forceinline__ float silu_mul(float g, float u) {
    const float t0 = -g * kLog2e, t = FAR ? fminf(t0, 126.f) : t0;
    const float lo = fabsf(t0) <= (FAR ? 512.f : 126.f) ? __builtin_fmaf(-g, kLog2e, -t0) - g * 1.92596299e-8f : 0.f;
    const float e0 = __builtin_amdgcn_exp2f(t), e = __builtin_fmaf(e0 * kLn2, lo, e0);
    const float r = g * __builtin_amdgcn_rcpf(1.f + e) * u;
    if (!FAR) return r;
    const float c = fminf(t0, 512.f), n = floorf(c), f = __builtin_amdgcn_exp2f(n - c);
    const int i = (int)n, h = i >> 1;
    return t0 > 126.f ? __builtin_ldexpf(g * __builtin_fmaf(f * -kLn2, lo, f), -h) * __builtin_ldexpf(u, h - i) : r;
}
/* Eight of them; the far form, which hardly any gates need, apart: in the way of every call it cost 4096 x 4096 0.3 of 4.9 us. */
static __device__ __forceinline__ void silu_mul_octet(float (&g)[8], const float (&u)[8]) {
    float least = g[0];
#pragma unroll
    for (int k = 1; k < 8; k++) least = fminf(least, g[k]);
    if (__builtin_expect(-least * kLog2e > 126.f, 0)) {
#pragma unroll
        for (int k = 0; k < 8; k++) g[k] = silu_mul<true>(g[k], u[k]);
    } else {
#pragma unroll
        for (int k = 0; k < 8; k++) g[k] = silu_mul<false>(g[k], u[k]);
    }
}
static __device__ __forceinline__ __amdgpu_buffer_rsrc_t rsrc(const void *p, unsigned n) { return __builtin_amdgcn_make_buffer_rsrc((void *)p, 0, n, 0x00027000); }
/* LDS writes of this wave's lanes are seen by its later reads (no other wave touches them). */
static __device__ __forceinline__ void wave_lds_fence() {
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
    __builtin_amdgcn_wave_barrier();
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
}

/* Eight values of type XTY at p as raw words, and those words as fp32. */
template <int XTY> struct XOct {
    uint4 w[XTY == 0 ? 2 : 1];
    __device__ __forceinline__ void load(const unsigned char *p) {
        w[0] = *(const uint4 *)p;
        if constexpr (XTY == 0) w[1] = *(const uint4 *)(p + 16);
    }
    __device__ __forceinline__ void up(float (&o)[8]) const {
        const unsigned *r = (const unsigned *)w;
        if constexpr (XTY == 0) {
#pragma unroll
            for (int i = 0; i < 8; i++) o[i] = flt(r[i]);
        } else if constexpr (XTY == 1) {
#pragma unroll
            for (int i = 0; i < 4; i++) o[2 * i] = XT<1>::up((unsigned short)r[i]), o[2 * i + 1] = XT<1>::up((unsigned short)(r[i] >> 16));
        } else {
#pragma unroll
            for (int i = 0; i < 4; i++) o[2 * i] = flt(r[i] << 16), o[2 * i + 1] = flt(r[i] & 0xFFFF0000u);
        }
    }
};

/* N scales or zero points of type STY as loaded: one by one, or at once from an address of that alignment (VEC; 16-bit ones then two to a
 * word). Where there are no zero points the buffer is empty and 0 comes back. */
template <int STY, int N, bool VEC> struct Scales {
    static constexpr int SB = STY == 0 ? 4 : 2;
    unsigned d[N];
    /* of blocks b .. b + N - 1 (of `sub` columns) of the matrix row that begins at value `row` */
    __device__ __forceinline__ void load(__amdgpu_buffer_rsrc_t r, unsigned row, int b, int sub, int cols, int gshift, int ng) {
        if constexpr (VEC) {
            const unsigned off = (row + min(b, ng - N)) * SB;
            if constexpr (N * SB == 16) {
                const auto v = __builtin_amdgcn_raw_buffer_load_b128(r, off, 0, 0);
                d[0] = v[0], d[1] = v[1], d[2] = v[2], d[3] = v[3];
            } else if constexpr (N * SB == 8) {
                const auto v = __builtin_amdgcn_raw_buffer_load_b64(r, off, 0, 0);
                d[0] = v[0], d[1] = v[1];
            } else {
                d[0] = __builtin_amdgcn_raw_buffer_load_b32(r, off, 0, 0);
            }
        } else {
#pragma unroll
            for (int k = 0; k < N; k++) {
                const unsigned off = (row + (min((b + k) * sub, cols - 1) >> gshift)) * SB;
                if constexpr (SB == 4) d[k] = __builtin_amdgcn_raw_buffer_load_b32(r, off, 0, 0);
                else d[k] = __builtin_amdgcn_raw_buffer_load_b16(r, off, 0, 0);
            }
        }
    }
    __device__ __forceinline__ float at(int k) const {
        if constexpr (STY == 0) return flt(d[k]);
        else return XT<STY>::up((unsigned short)(VEC && N > 1 ? d[k / 2] >> 16 * (k & 1) : d[k]));
    }
};

/* STY: type of the scales; T tokens (at most); P pieces; T * P <= 4; MP: more slices than waves */
template <int XTY, bool SW, int T, int P, int STY, int SUB, bool VEC, bool MP> __device__ __forceinline__ void g4q_body(const G4Args &a) {
    constexpr int BPC = 128 / SUB, XB = XTY == 0 ? 4 : 2, SB = STY == 0 ? 4 : 2;
    struct Item {
        uint4 q[4];
        Scales<STY, BPC, VEC> s, z;
    };
    constexpr bool QUAD = T == 1 && P > 1;  /* lane i of four takes octet i for all of them, exchanged through LDS */
    extern __shared__ __align__(16) unsigned char lds[]; /* QUAD: [wave][octet][kappa][g][piece] octets; then [group][wave][token][64] sums */
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), NW = a.nw;
    const int n = lane & 15, g = lane >> 4, s = blockIdx.y, groups = (a.rows + 15) >> 4;
    float *red = (float *)(lds + (QUAD ? NW * 4096 : 0));
    const int mat = a.sel ? a.sel[s] : s;
    auto store = [&](int t, int r, float v) {
        const size_t yo = ((size_t)s * a.m + t) * a.rows + r;
        ((typename XT<XTY>::raw *)a.y)[yo] = XT<XTY>::down(v);
    };
    if (mat < 0 || mat >= a.n_mat) { /* uniform over the block */
        for (int gr = blockIdx.x; gr < groups; gr += a.gx)
            if (threadIdx.x < 16 && gr * 16 + (int)threadIdx.x < a.rows)
                for (int t = 0; t < a.m; t++) store(t, gr * 16 + threadIdx.x, 0.f);
        return;
    }
    /* an item is a group of 16 rows in a pass over the waves' slices of 512 columns (one slice a wave and pass), pass by pass */
    const int ns = (a.cols + 511) >> 9, G = a.per - ((int)blockIdx.x >= a.full ? 1 : 0);
    const int items = MP ? (ns + NW - 1) / NW * G : G;

    /* activations of a pass: as loaded, then as pieces with their sums over the scale blocks */
    const int kappa = n >> 2, vi = n & 3, tok = T == 1 ? 0 : vi / P;
    const unsigned char *x = (const unsigned char *)a.x + (size_t)(s / a.share) * a.m * a.xstride * XB;
    constexpr int NO = QUAD ? 1 : 4;
    struct X {
        XOct<XTY> o[NO], u[SW ? NO : 1];
    } xn, xm; /* of the next pass to stage, of the one after */
    auto x_col = [&](int pass, int j) { return ((pass * NW + wave) * 4 + kappa) * 128 + octet_col<SUB>(QUAD ? vi : j, g); };
    auto x_load = [&](X &d, int pass) {
#pragma unroll
        for (int j = 0; j < NO; j++) {
            const int col = x_col(pass, j);
            const bool in = col < a.cols && tok < a.m;
            const unsigned char *p = x + ((size_t)(in ? tok : 0) * a.xstride + (in ? col : 0)) * XB;
            d.o[j].load(p);
            if constexpr (SW) d.u[j].load(p + (size_t)a.cols * XB);
        }
    };
    uint4 xa[4];
    float xs[BPC][T];
    auto stage = [&](int pass) {
        if constexpr (QUAD) {
            float f[8];
            xn.o[0].up(f);
            if constexpr (SW) {
                float u[8];
                xn.u[0].up(u);
                silu_mul_octet(f, u);
            }
            const bool in = x_col(pass, 0) < a.cols;
#pragma unroll
            for (int k = 0; k < 8; k++) f[k] = in ? f[k] : 0.f;
            uint4 *xl = (uint4 *)(lds + wave * 4096) + (kappa * 4 + g) * 4;
            /* cut, so that no piece exceeds the value; the last, of what is left, to nearest: exact but for SwiGLU's 24 bits in two
             * pieces, whose rest is below 2^-7 of the value's power of two and is held to 2^-16 of it */
#pragma unroll 1
            for (int p = 0; p < P - 1; p++) {
                xl[vi * 64 + p] = pack_octet(f);
#pragma unroll
                for (int k = 0; k < 8; k++) f[k] -= cut16(f[k]);
            }
            xl[vi * 64 + P - 1] = pack_octet_near(f);
#pragma unroll
            for (int p = P; p < 4; p++) xl[vi * 64 + p] = make_uint4(0, 0, 0, 0);
            wave_lds_fence();
#pragma unroll
            for (int j = 0; j < 4; j++) xa[j] = xl[j * 64 + vi];
            wave_lds_fence();
        } else {
#pragma unroll
            for (int j = 0; j < 4; j++) {
                float f[8];
                xn.o[j].up(f);
                const bool in = x_col(pass, j) < a.cols && (T > 1 ? tok < a.m : vi == 0);
#pragma unroll
                for (int k = 0; k < 8; k++) {
                    f[k] = in ? f[k] : 0.f;
                    if constexpr (P == 2) f[k] = vi & 1 ? f[k] - cut16(f[k]) : f[k];
                }
                xa[j] = pack_octet(f);
            }
        }
        const unsigned one = 0x3F803F80u;
        const bf16x8 ones = __builtin_bit_cast(bf16x8, make_uint4(one, one, one, one));
#pragma unroll
        for (int b = 0; b < BPC; b++) {
            f32x4 d = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int j = b * (4 / BPC); j < (b + 1) * (4 / BPC); j++) d = mfma(xa[j], ones, d);
#pragma unroll
            for (int t = 0; t < T; t++) {
                xs[b][t] = d[t * P];
#pragma unroll
                for (int p = 1; p < P; p++) xs[b][t] += d[t * P + p];
            }
        }
    };

    const float zbase = a.zeros ? 16.f : 24.f;
    const unsigned rowb = a.cols >> 1;
    unsigned vo[4];
#pragma unroll
    for (int u = 0; u < 4; u++) vo[u] = (4 * u + (n >> 2)) * rowb + ((n + u) & 3) * 64 + g * 16;
    const int us = (g - n) & 3, myrow = 4 * us + (n >> 2); /* the step whose result this lane keeps, and its row */
    const unsigned bytes = a.rows * rowb, sbytes = a.rows * a.ng * SB; /* of the matrix: below 4 GiB */
    const unsigned char *w0 = a.codes + (size_t)mat * bytes, *s0 = (const unsigned char *)a.scales + (size_t)mat * sbytes,
                        *z0 = (const unsigned char *)a.zeros + (size_t)mat * sbytes;
    auto load = [&](Item &it, bool there, int pass, int gi) { /* loads come back in order: scales before the codes they belong to */
        const int gr = (int)blockIdx.x + gi * a.gx, sl = (MP ? pass * NW : 0) + wave;
        there = there && sl < ns;
        const auto rq = rsrc(w0, there ? bytes : 0), rs = rsrc(s0, there ? sbytes : 0), rz = rsrc(z0, there && a.zeros ? sbytes : 0);
        const unsigned row = (gr * 16 + myrow) * a.ng;
        it.s.load(rs, row, (sl * 4 + g) * BPC, SUB, a.cols, a.gshift, a.ng);
        it.z.load(rz, row, (sl * 4 + g) * BPC, SUB, a.cols, a.gshift, a.ng);
        const unsigned go = gr * 16 * rowb + sl * 256;
#pragma unroll
        for (int u = 0; u < 4; u++) it.q[u] = __builtin_bit_cast(uint4, __builtin_amdgcn_raw_buffer_load_b128(rq, vo[u] + go, 0, 2 /* nt */));
    };
    unsigned mask = 0x00780078u;
    asm volatile("" : "+v"(mask));
    auto work = [&](Item &it, int pass, int gi) {
        float keep[BPC][T * P];
#pragma unroll
        for (int u = 0; u < 4; u++) {
            spread<SUB>(it.q[u]);
            const unsigned qw[4] = {it.q[u].x, it.q[u].y, it.q[u].z, it.q[u].w};
#pragma unroll
            for (int b = 0; b < BPC; b++) {
                f32x4 d = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
                for (int j = b * (4 / BPC); j < (b + 1) * (4 / BPC); j++) d = mfma(xa[j], unpack(qw[j], mask), d);
#pragma unroll
                for (int i = 0; i < T * P; i++) keep[b][i] = u == 0 || u == us ? d[i] : keep[b][i];
            }
        }
#pragma unroll
        for (int t = 0; t < T; t++) {
            float tot = 0.f;
#pragma unroll
            for (int b = 0; b < BPC; b++) {
                const float sc = it.s.at(b), zo = zbase + it.z.at(b);
                const bool in = (((MP ? pass * NW : 0) + wave) * 4 + g) * 128 + b * SUB < a.cols;
                float d = keep[b][t * P];
#pragma unroll
                for (int p = 1; p < P; p++) d += keep[b][t * P + p];
                const float v = sc * __builtin_fmaf(-zo, xs[b][t], d);
                tot += in ? v : 0.f;
            }
            float *to = &red[((gi * NW + wave) * T + t) * 64 + myrow * 4 + g];
            *to = MP && pass ? *to + tot : tot;
        }
    };
    Item A, B;
    int lp = 0, lg = 0, wp = 0, wg = 0; /* pass and group of the next item to load, to multiply */
    auto step = [&](int &p, int &gi) {
        if (++gi == G) gi = 0, p++;
    };
    x_load(xn, 0);
    if (MP) x_load(xm, 1);
    __builtin_amdgcn_sched_barrier(0); /* in this order */
    load(A, true, lp, lg);
    step(lp, lg);
    load(B, 1 < items, lp, lg);
    step(lp, lg);
    if (!MP) stage(0);
    for (int i = 0;; i += 2) { /* no prologue or tail of their own: code is fetched cold at every launch, 15..20 ns a 64-byte line */
        if (MP && wg == 0) {
            stage(wp);
            xn = xm;
            x_load(xm, wp + 2);
        }
        work(A, wp, wg);
        if (i + 1 >= items) break;
        load(A, i + 2 < items, lp, lg);
        step(lp, lg);
        step(wp, wg);
        if (MP && wg == 0) {
            stage(wp);
            xn = xm;
            x_load(xm, wp + 2);
        }
        work(B, wp, wg);
        if (i + 2 >= items) break;
        load(B, i + 3 < items, lp, lg);
        step(lp, lg);
        step(wp, wg);
    }
    __syncthreads();
    for (int gi = wave; gi < G; gi += NW) { /* the waves' partial results, added in wave order */
        const int r = ((int)blockIdx.x + gi * a.gx) * 16 + (lane >> 2);
#pragma unroll
        for (int t = 0; t < T; t++) {
            float v = red[(gi * NW * T + t) * 64 + lane];
            for (int w = 1; w < NW; w++) v += red[((gi * NW + w) * T + t) * 64 + lane];
            v += flt(__builtin_amdgcn_mov_dpp(bits(v), 0xB1, 0xf, 0xf, true)); /* quad lanes 1 0 3 2 */
            v += flt(__builtin_amdgcn_mov_dpp(bits(v), 0x4E, 0xf, 0xf, true)); /* quad lanes 2 3 0 1 */
            if (r < a.rows && (lane & 3) == 0 && (T == 1 || t < a.m)) store(t, r, v);
        }
    }
}

#ifndef LE_G4_STY
#define LE_G4_STY 1 /* a code object for each type of scales */
#endif
#define LE_G4_CAT2(a, b) a##b
#define LE_G4_CAT(a, b) LE_G4_CAT2(a, b)
#define LE_G4_S LE_G4_CAT(_s, LE_G4_STY)
#define LE_G4_KERNEL(BLOCK, NAME, BODY) extern "C" __global__ void __launch_bounds__(BLOCK) LE_G4_CAT(NAME, LE_G4_S)(G4Args a) { BODY(a); }
/* F(suffix, SUB, VEC, ...) for all scale blocks */
#define LE_G4_SUBS(F, ...) F(b32, 32, false, __VA_ARGS__) F(b32v, 32, true, __VA_ARGS__) F(b64, 64, false, __VA_ARGS__) F(b64v, 64, true, __VA_ARGS__) \
    F(b128, 128, false, __VA_ARGS__)
#define LE_G4Q1(B, SUB, VEC, NAME, XTY, SW, T, P) \
    LE_G4_KERNEL(512, le_g4q_##NAME##_##B, (g4q_body<XTY, SW, T, P, LE_G4_STY, SUB, VEC, false>)) \
    LE_G4_KERNEL((T == 1 || SUB >= 64 ? 1024 : 512), le_g4q_##NAME##_##B##_mp, (g4q_body<XTY, SW, T, P, LE_G4_STY, SUB, VEC, true>))
LE_G4_SUBS(LE_G4Q1, f32, 0, false, 1, 3)
LE_G4_SUBS(LE_G4Q1, f16, 1, false, 1, 2)
LE_G4_SUBS(LE_G4Q1, bf16, 30, false, 1, 1)
LE_G4_SUBS(LE_G4Q1, f32w, 0, true, 1, 3)
LE_G4_SUBS(LE_G4Q1, f16w, 1, true, 1, 2)
LE_G4_SUBS(LE_G4Q1, bf16w, 30, true, 1, 2)
LE_G4_SUBS(LE_G4Q1, f16t2, 1, false, 2, 2)
LE_G4_SUBS(LE_G4Q1, bf16t4, 30, false, 4, 1)

/* ---- more tokens: activations laid out by a launch of their own ----
 *
 * le_g4x_*: the activations as MFMA fragments in the workspace, 16 bytes a lane: up to 12 virtual rows (tokens times pieces, a.na sets of
 * four) as le_g4t_* takes them, [slice of 512 columns][MFMA j][set][lane]; more tokens as le_g4m_* does, tiles of 16,
 * [chunk of 128 columns][MFMA j][piece][lane group][token]. SwiGLU and the cut into pieces are thus done once a launch and not once a block. The pieces are
 * fp16 here, of the chunk's activations times the power of two that brings the largest to [2^14, 2^15): one piece holds bf16 and fp16, two hold
 * 22 bits (fp32 and SwiGLU's result; what is cut off is below 2^-23 of the value, or 2^-39 of the chunk's largest), where bf16
 * would take three. Beside them the powers' reciprocals, [chunk][16 tokens]. A thread takes an octet of a token. */
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));

template <int XTY, bool SW, int P, int SUB> __device__ __forceinline__ void g4x_body(const G4Args &a) {
    constexpr int XB = XTY == 0 ? 4 : 2;
    const int nc = (a.cols + 127) >> 7, no = nc * 16;
    const int oc = blockIdx.x * 256 + threadIdx.x, tok = blockIdx.y % a.m, set = blockIdx.y / a.m;
    if (oc >= no) return; /* whole chunks: the shuffles below stay within one */
    const int tile = tok >> 4, tm = min(16, a.m - tile * 16);
    const bool in = oc * 8 < a.cols;
    const unsigned char *x = (const unsigned char *)a.x + (((size_t)set * a.m + tok) * a.xstride + (in ? oc * 8 : 0)) * XB;
    XOct<XTY> o, uo;
    o.load(x);
    if constexpr (SW) uo.load(x + (size_t)a.cols * XB);
    float f[8];
    o.up(f);
    if constexpr (SW) {
        float u[8];
        uo.up(u);
        silu_mul_octet(f, u);
    }
    float big = 0.f;
#pragma unroll
    for (int k = 0; k < 8; k++) {
        f[k] = in ? f[k] : 0.f;
        big = fmaxf(big, fabsf(f[k]));
    }
#pragma unroll
    for (int d = 1; d < 16; d <<= 1) big = fmaxf(big, __shfl_xor(big, d));
    /* 2^(14 - exponent of big), at most 2^126; infinite or NaN values stay what they are */
    const int e = min(141 - (int)(bits(big) >> 23), 126);
    const float up = flt((unsigned)(e + 127) << 23), down = flt((unsigned)(127 - e) << 23);
    unsigned char *ws = (unsigned char *)a.ws + (size_t)set * a.ws_set;
    /* where octet o of a chunk goes: MFMA j, lane group g (octet_col's inverse) */
    const int hi = (oc >> 2) & 3, lo = oc & 3;
    const int j = SUB == 128 ? lo : SUB == 64 ? 2 * (hi >> 1) + (lo & 1) : hi, g = SUB == 128 ? hi : SUB == 64 ? (hi & 1) + 2 * (lo >> 1) : lo;
    uint4 *frag = (uint4 *)ws + (size_t)no * P * tile * 16 + ((size_t)((oc >> 4) * 4 + j) * P * 4 + g) * tm + (tok & 15);
    int step = 4 * tm; /* from piece to piece */
    if (a.na) {
        const int v = tok * P; /* a token's pieces lie in one set: sets are four rows, P is 1 or 2 */
        frag = (uint4 *)ws + ((size_t)((oc >> 6) * 4 + j) * a.na + (v >> 2)) * 64 + g * 16 + ((oc >> 4) & 3) * 4 + (v & 3);
        step = 1;
    }
#pragma unroll
    for (int k = 0; k < 8; k++) f[k] *= up;
#pragma unroll
    for (int p = 0; p < P; p++) {
        _Float16 h[8];
#pragma unroll
        for (int k = 0; k < 8; k++) {
            h[k] = (_Float16)f[k];
            f[k] -= (float)h[k];
        }
        auto two = [&](int k) { return __builtin_bit_cast(unsigned, (f16x2){h[k], h[k + 4]}); };
        frag[p * step] = make_uint4(two(0), two(1), two(2), two(3));
    }
    if ((oc & 15) == 0) {
        float *downs = (float *)(ws + a.ws_downs) + ((size_t)tile * nc + (oc >> 4)) * 16;
        downs[tok & 15] = down;
        if (tok == a.m - 1)
            for (int t = tm; t < 16; t++) downs[t] = 0.f;
    }
}

/* Eight codes as fp16 16 + code (k: 0x03C003C0, as in unpack). */
static __device__ __forceinline__ f16x8 unpack16(unsigned q, unsigned k) {
    const unsigned o = 0x4C004C00u; /* 16; a step of the last place is 2^-6 */
    return __builtin_bit_cast(f16x8, make_uint4(((q << 6) & k) | o, ((q << 2) & k) | o, ((q >> 2) & k) | o, ((q >> 6) & k) | o));
}
static __device__ __forceinline__ f32x4 mfma16(const uint4 &a, const f16x8 &b, const f32x4 &c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, a), b, c, 0, 0, 0);
}

/* le_g4t_*: le_g4q_*'s layout with NA sets of four virtual rows, from the workspace; K in segments of a block's waves where it is
 * longer than they hold, whose partial results le_g4s adds. Against the layout of le_g4m_* it has fewer vector instructions (a lane
 * applies scale and zero point to one K part of one row, not to every one) and longer runs of a row's codes, for MFMAs that a few
 * tokens leave idle. */
template <int NA, int P, int STY, int SUB, bool VEC> __device__ __forceinline__ void g4t_body(const G4Args &a) {
    constexpr int BPC = 128 / SUB, T = 4 / P, NT = NA * T, SB = STY == 0 ? 4 : 2;
    struct Item {
        uint4 q[4];
        Scales<STY, BPC, VEC> s, z;
    };
    extern __shared__ __align__(16) unsigned char lds[];
    float *red = (float *)lds; /* [group][wave][token][64] */
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), NW = a.nw;
    const int n = lane & 15, g = lane >> 4, s = blockIdx.y, seg = blockIdx.z, groups = (a.rows + 15) >> 4;
    const int mat = a.sel ? a.sel[s] : s;
    auto store = [&](int t, int r, float v) {
        const size_t yo = ((size_t)s * a.m + t) * a.rows + r;
        if (a.segs > 1) a.part[(size_t)seg * a.total + yo] = v;
        else if (a.xty == 0) ((float *)a.y)[yo] = v;
        else ((unsigned short *)a.y)[yo] = a.xty == 1 ? XT<1>::down(v) : XT<30>::down(v);
    };
    if (mat < 0 || mat >= a.n_mat) { /* uniform over the block */
        for (int gr = blockIdx.x; gr < groups; gr += a.gx)
            if (threadIdx.x < 16 && gr * 16 + (int)threadIdx.x < a.rows)
                for (int t = 0; t < a.m; t++) store(t, gr * 16 + threadIdx.x, 0.f);
        return;
    }
    const int nc = (a.cols + 127) >> 7, ns = (nc + 3) >> 2, G = a.per - ((int)blockIdx.x >= a.full ? 1 : 0);
    const int sl = seg * NW + wave, slc = min(sl, ns - 1); /* a slice that is not there: no codes are read, and its result is left out */
    const unsigned char *ws = (const unsigned char *)a.ws + (size_t)(s / a.share) * a.ws_set;
    const uint4 *frag = (const uint4 *)ws + (size_t)slc * 4 * NA * 64 + lane;
    const float *downs = (const float *)(ws + a.ws_downs) + (size_t)min(slc * 4 + g, nc - 1) * 16;
    uint4 x[NA][4];
    float down[NT];
#pragma unroll
    for (int j = 0; j < 4; j++)
#pragma unroll
        for (int v = 0; v < NA; v++) x[v][j] = frag[(j * NA + v) * 64];
#pragma unroll
    for (int t = 0; t < NT; t++) down[t] = downs[t];
    __builtin_amdgcn_sched_barrier(0); /* loads return in order: these first */

    const float zbase = a.zeros ? 16.f : 24.f;
    const unsigned rowb = a.cols >> 1, bytes = a.rows * rowb, sbytes = a.rows * a.ng * SB; /* of the matrix: below 4 GiB */
    unsigned vo[4];
#pragma unroll
    for (int u = 0; u < 4; u++) vo[u] = (4 * u + (n >> 2)) * rowb + sl * 256 + ((n + u) & 3) * 64 + g * 16;
    const int us = (g - n) & 3, myrow = 4 * us + (n >> 2); /* the step whose result this lane keeps, and its row */
    const unsigned char *w0 = a.codes + (size_t)mat * bytes, *s0 = (const unsigned char *)a.scales + (size_t)mat * sbytes,
                        *z0 = (const unsigned char *)a.zeros + (size_t)mat * sbytes;
    auto load = [&](Item &it, int gi) {
        const int gr = (int)blockIdx.x + gi * a.gx;
        const bool there = gi < G && sl < ns;
        const auto rq = rsrc(w0, there ? bytes : 0), rs = rsrc(s0, there ? sbytes : 0), rz = rsrc(z0, there && a.zeros ? sbytes : 0);
        const unsigned row = (gr * 16 + myrow) * a.ng;
        it.s.load(rs, row, (sl * 4 + g) * BPC, SUB, a.cols, a.gshift, a.ng);
        it.z.load(rz, row, (sl * 4 + g) * BPC, SUB, a.cols, a.gshift, a.ng);
        const unsigned go = gr * 16 * rowb;
#pragma unroll
        for (int u = 0; u < 4; u++) it.q[u] = __builtin_bit_cast(uint4, __builtin_amdgcn_raw_buffer_load_b128(rq, vo[u] + go, 0, 2 /* nt */));
    };
    unsigned mask = 0x03C003C0u;
    asm volatile("" : "+v"(mask));
    auto work = [&](Item &it, int gi, const float (&xs)[BPC][NT]) {
        float keep[BPC][NA * 4];
#pragma unroll
        for (int u = 0; u < 4; u++) {
            spread<SUB>(it.q[u]);
            const unsigned qw[4] = {it.q[u].x, it.q[u].y, it.q[u].z, it.q[u].w};
#pragma unroll
            for (int b = 0; b < BPC; b++) {
                f32x4 d[NA];
#pragma unroll
                for (int v = 0; v < NA; v++) d[v] = (f32x4){0.f, 0.f, 0.f, 0.f};
#pragma unroll
                for (int j = b * (4 / BPC); j < (b + 1) * (4 / BPC); j++) {
                    const f16x8 w = unpack16(qw[j], mask);
#pragma unroll
                    for (int v = 0; v < NA; v++) d[v] = mfma16(x[v][j], w, d[v]);
                }
#pragma unroll
                for (int i = 0; i < NA * 4; i++) keep[b][i] = u == 0 || u == us ? d[i / 4][i % 4] : keep[b][i];
            }
        }
        float tot[NT] = {};
#pragma unroll
        for (int b = 0; b < BPC; b++) {
            const float sc = it.s.at(b), zo = zbase + it.z.at(b);
            const bool in = (sl * 4 + g) * 128 + b * SUB < a.cols;
#pragma unroll
            for (int t = 0; t < NT; t++) {
                const float d = P == 2 ? keep[b][2 * t] + keep[b][2 * t + 1] : keep[b][t], v = sc * __builtin_fmaf(-zo, xs[b][t], d);
                tot[t] += in ? v : 0.f;
            }
        }
#pragma unroll
        for (int t = 0; t < NT; t++) red[((gi * NW + wave) * NT + t) * 64 + myrow * 4 + g] = tot[t] * down[t];
    };
    Item A, B;
    load(A, 0);
    load(B, 1);
    float xs[BPC][NT]; /* sums of the activations over the scale blocks, where the results lie: the same MFMAs with codes of 1 */
    {
        const unsigned one = 0x3C003C00u;
        const f16x8 ones = __builtin_bit_cast(f16x8, make_uint4(one, one, one, one));
#pragma unroll
        for (int b = 0; b < BPC; b++)
#pragma unroll
            for (int v = 0; v < NA; v++) {
                f32x4 d = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
                for (int j = b * (4 / BPC); j < (b + 1) * (4 / BPC); j++) d = mfma16(x[v][j], ones, d);
#pragma unroll
                for (int t = 0; t < T; t++) xs[b][v * T + t] = P == 2 ? d[(2 * t) & 3] + d[(2 * t + 1) & 3] : d[t];
            }
    }
    for (int gi = 0;; gi += 2) {
        work(A, gi, xs);
        if (gi + 1 >= G) break;
        load(A, gi + 2);
        work(B, gi + 1, xs);
        if (gi + 2 >= G) break;
        load(B, gi + 3);
    }
    __syncthreads();
    for (int i = wave; i < G * NT; i += NW) { /* the waves' partial results, added in wave order */
        const int gi = i / NT, t = i % NT, r = ((int)blockIdx.x + gi * a.gx) * 16 + (lane >> 2);
        if (t >= a.m) continue;
        float v = red[(gi * NW * NT + t) * 64 + lane];
        for (int w = 1; w < NW; w++) v += red[((gi * NW + w) * NT + t) * 64 + lane];
        v += flt(__builtin_amdgcn_mov_dpp(bits(v), 0xB1, 0xf, 0xf, true)); /* quad lanes 1 0 3 2 */
        v += flt(__builtin_amdgcn_mov_dpp(bits(v), 0x4E, 0xf, 0xf, true)); /* quad lanes 2 3 0 1 */
        if (r < a.rows && (lane & 3) == 0) store(t, r, v);
    }
}

/* le_g4m_*: 16 tokens as the rows of v_mfma_f32_16x16x32_f16, 16 weight rows as its columns (codes as fp16 16 + code): lane (n, g) loads
 * 16 bytes of row n at 32 g of a chunk. A wave keeps the fragments of a slice of CS chunks in registers and goes over the block's row
 * groups with it, as above. Where K has more chunks than the waves of a block hold, it is cut into segments, each a block's own, whose
 * partial results le_g4s adds: with passes instead (as le_g4q_*), every block of a long K reads all fragments for its few
 * rows, one pass's at a time (4096 x 14336, five tokens: 29 us). The scales of
 * an item are loaded once by the lane groups together and passed between them: loaded by each lane group they were a third of the
 * time (14336 x 4096 bf16, five tokens 18.4 us, 12.6 without those loads). 14336 x 4096 fp32, groups of 128: 16 tokens 17.0 us, 32 22.8, 64 34.7. */
template <int P, int STY, int SUB, bool VEC, int CS> __device__ __forceinline__ void g4m_body(const G4Args &a) {
    constexpr int SB = STY == 0 ? 4 : 2, BPC = 128 / SUB, NL = CS * BPC / 4; /* NL: of an item's scale blocks, a lane's to load */
    struct Item {
        uint4 q[CS];
        Scales<STY, NL, VEC && (NL > 1)> s, z;
    };
    extern __shared__ __align__(16) unsigned char lds[];
    f32x4 *red = (f32x4 *)lds; /* [group][wave][64] */
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), NW = a.nw;
    const int n = lane & 15, g = lane >> 4, s = blockIdx.y, seg = blockIdx.z % a.segs, tile = blockIdx.z / a.segs, t0 = tile * 16, tm = min(16, a.m - t0), groups = (a.rows + 15) >> 4;
    const int mat = a.sel ? a.sel[s] : s;
    auto store = [&](int t, int r, float v) {
        const size_t yo = ((size_t)s * a.m + t0 + t) * a.rows + r;
        if (a.segs > 1) a.part[(size_t)seg * a.total + yo] = v;
        else if (a.xty == 0) ((float *)a.y)[yo] = v;
        else ((unsigned short *)a.y)[yo] = a.xty == 1 ? XT<1>::down(v) : XT<30>::down(v);
    };
    if (mat < 0 || mat >= a.n_mat) { /* uniform over the block */
        for (int gr = blockIdx.x; gr < groups; gr += a.gx)
            if (threadIdx.x < 16 && gr * 16 + (int)threadIdx.x < a.rows)
                for (int t = 0; t < tm; t++) store(t, gr * 16 + threadIdx.x, 0.f);
        return;
    }
    const int nc = (a.cols + 127) >> 7, G = a.per - ((int)blockIdx.x >= a.full ? 1 : 0), c0 = (seg * NW + wave) * CS;
    const unsigned char *ws = (const unsigned char *)a.ws + (size_t)(s / a.share) * a.ws_set;
    const uint4 *frag = (const uint4 *)ws + (size_t)nc * 16 * P * t0 + g * tm + min(n, tm - 1);
    const f32x4 *downs = (const f32x4 *)(ws + a.ws_downs) + (size_t)tile * nc * 4 + g;
    uint4 x[CS][4][P];
    f32x4 down[CS];
#pragma unroll
    for (int c = 0; c < CS; c++) {
        const int cc = min(c0 + c, nc - 1); /* a chunk that is not there: its result is left out */
#pragma unroll
        for (int j = 0; j < 4; j++)
#pragma unroll
            for (int p = 0; p < P; p++) x[c][j][p] = frag[(((size_t)cc * 4 + j) * P + p) * 4 * tm];
        down[c] = downs[cc * 4];
    }
    __builtin_amdgcn_sched_barrier(0); /* loads return in order: these first */
    const float zbase = a.zeros ? 16.f : 24.f;
    const unsigned rowb = a.cols >> 1, bytes = a.rows * rowb, sbytes = a.rows * a.ng * SB; /* of the matrix: below 4 GiB */
    const unsigned char *w0 = a.codes + (size_t)mat * bytes, *s0 = (const unsigned char *)a.scales + (size_t)mat * sbytes,
                        *z0 = (const unsigned char *)a.zeros + (size_t)mat * sbytes;
    const unsigned vo = n * rowb + g * 16;
    auto load = [&](Item &it, int gi) {
        const int gr = (int)blockIdx.x + gi * a.gx;
        const bool there = gi < G;
        const auto rq = rsrc(w0, there ? bytes : 0), rs = rsrc(s0, there ? sbytes : 0), rz = rsrc(z0, there && a.zeros ? sbytes : 0);
        const int b0 = c0 * BPC + g * NL;
        const unsigned row = (gr * 16 + n) * a.ng;
        it.s.load(rs, row, b0, SUB, a.cols, a.gshift, a.ng);
        it.z.load(rz, row, b0, SUB, a.cols, a.gshift, a.ng);
        const unsigned go = gr * 16 * rowb + c0 * 64;
#pragma unroll
        for (int c = 0; c < CS; c++)
            it.q[c] = __builtin_bit_cast(uint4, __builtin_amdgcn_raw_buffer_load_b128(rq, c0 + c < nc ? vo + go + c * 64 : 0xFFFFFFF0u, 0, 2 /* nt */));
    };
    unsigned mask = 0x03C003C0u;
    asm volatile("" : "+v"(mask));
    auto work = [&](Item &it, int gi, const f32x4 (&sum)[CS][BPC]) {
        float sc[NL], zo[NL]; /* this lane's blocks, scale and 16 + zero point */
#pragma unroll
        for (int k = 0; k < NL; k++) {
            sc[k] = it.s.at(k);
            zo[k] = zbase + it.z.at(k);
        }
        f32x4 tot = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int c = 0; c < CS; c++) {
            spread<SUB>(it.q[c]);
            const unsigned qw[4] = {it.q[c].x, it.q[c].y, it.q[c].z, it.q[c].w};
            f32x4 part = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int b = 0; b < BPC; b++) {
                f32x4 d = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
                for (int j = b * (4 / BPC); j < (b + 1) * (4 / BPC); j++) {
                    const f16x8 w = unpack16(qw[j], mask);
#pragma unroll
                    for (int p = 0; p < P; p++) d = mfma16(x[c][j][p], w, d);
                }
                const int at = c * BPC + b, from = ((at / NL) * 16 + n) * 4;
                const float s1 = flt(__builtin_amdgcn_ds_bpermute(from, bits(sc[at % NL]))), z1 = flt(__builtin_amdgcn_ds_bpermute(from, bits(zo[at % NL])));
                const bool in = (c0 + c) * 128 + b * SUB < a.cols;
#pragma unroll
                for (int i = 0; i < 4; i++) {
                    const float v = s1 * __builtin_fmaf(-z1, sum[c][b][i], d[i]);
                    part[i] += in ? v : 0.f;
                }
            }
#pragma unroll
            for (int i = 0; i < 4; i++) tot[i] = __builtin_fmaf(part[i], down[c][i], tot[i]);
        }
        red[(gi * NW + wave) * 64 + lane] = tot;
    };
    Item A, B;
    load(A, 0);
    load(B, 1);
    f32x4 sum[CS][BPC]; /* of the activations over the scale blocks, where the results lie: the same MFMAs with codes of 1 */
    {
        const unsigned one = 0x3C003C00u;
        const f16x8 ones = __builtin_bit_cast(f16x8, make_uint4(one, one, one, one));
#pragma unroll
        for (int c = 0; c < CS; c++)
#pragma unroll
            for (int b = 0; b < BPC; b++) {
                f32x4 d = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
                for (int j = b * (4 / BPC); j < (b + 1) * (4 / BPC); j++)
#pragma unroll
                    for (int p = 0; p < P; p++) d = mfma16(x[c][j][p], ones, d);
                sum[c][b] = d;
            }
    }
    for (int gi = 0;; gi += 2) {
        work(A, gi, sum);
        if (gi + 1 >= G) break;
        load(A, gi + 2);
        work(B, gi + 1, sum);
        if (gi + 2 >= G) break;
        load(B, gi + 3);
    }
    __syncthreads();
    for (int gi = wave; gi < G; gi += NW) { /* the waves' partial results, added in wave order */
        const int r = ((int)blockIdx.x + gi * a.gx) * 16 + n;
        f32x4 v = red[gi * NW * 64 + lane];
        for (int w = 1; w < NW; w++) v += red[(gi * NW + w) * 64 + lane];
#pragma unroll
        for (int i = 0; i < 4; i++)
            if (r < a.rows && g * 4 + i < tm) store(g * 4 + i, r, v[i]);
    }
}

/* 16 waves, which leave each 128 registers: one set, and two at scale blocks of 64 and more; 12 waves (168): two sets of two pieces at 32, three
 * at 64 and more; two sets of one piece at 64 (143 registers)
 * as a kernel of its own for long rows, which spills a few (14336 x 4096 bf16, 8 tokens 14.8 us, with spills 16.2; 5120 x 5120, 6
 * tokens, in two segments of eight waves 15.0, in one of ten 11.4) */
#define LE_G4T1(B, SUB, VEC, NA, P) \
    LE_G4_KERNEL((NA == 1 || (NA == 2 && (SUB == 128 || (SUB == 64 && P == 2))) ? 1024 : (NA == 3 && SUB >= 64) || (NA == 2 && P == 2) ? 768 : 512), le_g4t_n##NA##_p##P##_##B, (g4t_body<NA, P, LE_G4_STY, SUB, VEC>))
LE_G4_KERNEL(1024, le_g4t_n2_p1_b64_w, (g4t_body<2, 1, LE_G4_STY, 64, false>)) LE_G4_KERNEL(1024, le_g4t_n2_p1_b64v_w, (g4t_body<2, 1, LE_G4_STY, 64, true>))
LE_G4_SUBS(LE_G4T1, 1, 1) LE_G4_SUBS(LE_G4T1, 2, 1) LE_G4_SUBS(LE_G4T1, 1, 2) LE_G4_SUBS(LE_G4T1, 2, 2) LE_G4_SUBS(LE_G4T1, 3, 2)
#define LE_G4M1(B, SUB, VEC, P) LE_G4_KERNEL(512, le_g4m_p##P##_##B, (g4m_body<P, LE_G4_STY, SUB, VEC, (P == 2 && SUB == 32 ? 2 : 4)>))
LE_G4_SUBS(LE_G4M1, 1) LE_G4_SUBS(LE_G4M1, 2)

#if LE_G4_STY == 1 /* once */
#define LE_G4X(NAME, XTY, SW, P)                                                                                     \
    extern "C" __global__ void __launch_bounds__(256) le_g4x_##NAME##_b32(G4Args a) { g4x_body<XTY, SW, P, 32>(a); } \
    extern "C" __global__ void __launch_bounds__(256) le_g4x_##NAME##_b64(G4Args a) { g4x_body<XTY, SW, P, 64>(a); } \
    extern "C" __global__ void __launch_bounds__(256) le_g4x_##NAME##_b128(G4Args a) { g4x_body<XTY, SW, P, 128>(a); }
LE_G4X(f32, 0, false, 2) LE_G4X(f16, 1, false, 1) LE_G4X(bf16, 30, false, 1) LE_G4X(f32w, 0, true, 2) LE_G4X(f16w, 1, true, 2) LE_G4X(bf16w, 30, true, 2)

/* le_g4s: the segments' partial results added in their order and rounded, a value a thread. */
extern "C" __global__ void __launch_bounds__(256) le_g4s(G4Args a) {
    const size_t i = (size_t)blockIdx.x * 256 + threadIdx.x, n = (size_t)a.total;
    if (i >= n) return;
    float v = a.part[i];
#pragma unroll 4
    for (int s = 1; s < a.segs; s++) v += a.part[(size_t)s * n + i];
    if (a.xty == 0) ((float *)a.y)[i] = v;
    else ((unsigned short *)a.y)[i] = a.xty == 1 ? XT<1>::down(v) : XT<30>::down(v);
}
#endif
