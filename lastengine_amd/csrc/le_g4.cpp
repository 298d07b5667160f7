/* Host side of the matrix-vector products with 4-bit codes and group scales (le_matvec_g4, include/le_qmm.h): argument
 * checks and launch shapes. */
#include <algorithm>
#include <cstdint>
#include <cstdio>

#include "le_ctx.h"
#include "le_g4_args.h"

namespace {

int type_bytes(int ty) { return ty == LE_F32 ? 4 : ty == LE_F16 || ty == LE_BF16 ? 2 : 0; }
bool aligned(const void *p, unsigned n) { return ((uintptr_t)p & (n - 1)) == 0; }

/* (Times in this file: graph replays over 700 MB of weights, which no cache holds.)
 * One launch: bf16 pieces that hold an activation: 24 bits of fp32 in three, 11 of fp16 in two. SwiGLU's fp32 result: three, or the 16
 * bits of two, rounded, where the output is rounded to 11 or 8. */
int pieces(int xtype, int swiglu) { return xtype == LE_F32 ? 3 : xtype == LE_F16 || swiglu ? 2 : 1; }
/* Columns that a scale is applied to at a time. */
int scale_block(const le_g4 *w) { return w->group % 128 == 0 || w->group == w->cols ? 128 : w->group % 64 == 0 ? 64 : 32; }
/* ... and the tokens of a slot that it takes (le_g4q_*, four virtual rows). More need the activations laid out in the workspace, as ... */
int most_tokens(int xtype, int swiglu) { return swiglu ? 1 : 4 / pieces(xtype, 0); }
/* ... fp16 pieces (le_g4x_*, le_g4m_*). */
int pieces16(int xtype, int swiglu) { return xtype == LE_F32 || swiglu ? 2 : 1; }
/* le_g4t_*: sets of four virtual rows, up to two, or three of two pieces a token; 0: le_g4m_*, whose rows are 16 tokens. 14336 x 4096,
 * le_g4t_* / le_g4m_* in us, fp32, groups of 32, 64, 128: 2 tokens (one set) 12.5 / 18.9, 11.9 / 18.3, 11.1 / 15.8; 4 (two) 15.2 / 19.1,
 * 13.8 / 18.1, 13.3 / 16.2; 5 (three) 18.0 / 19.4, 16.1 / 18.1, 15.7 / 16.1; 8 (four) 20.6 / 19.7, 18.4 / 18.1, 17.2 / 16.2; bf16, 8
 * tokens (two) 16.5 / 17.9, 14.9 / 16.5, 14.2 / 14.6, 9 (three) 22.3 / 18.0, 19.5 / 16.6, 18.3 / 14.7. */
int row_sets(int xtype, int swiglu, int m) {
    const int p = pieces16(xtype, swiglu), na = (m * p + 3) / 4;
    return na <= 2 || (na == 3 && p == 2) ? na : 0;
}
/* Bytes of one set of activations: fragments, powers of two. */
size_t frag_bytes(int xtype, int swiglu, int m, int cols) {
    const size_t nc = (size_t)(cols + 127) / 128;
    if (const int na = row_sets(xtype, swiglu, m)) return (nc + 3) / 4 * 4096 * na;
    return nc * 256 * pieces16(xtype, swiglu) * m;
}
size_t tile_floats(int m, int cols) { return (size_t)((m + 15) / 16) * ((cols + 127) / 128) * 16; }
size_t set_bytes(int xtype, int swiglu, int m, int cols) { return frag_bytes(xtype, swiglu, m, cols) + tile_floats(m, cols) * 4; }
/* 128-column chunks that a wave keeps (le_g4m_*: two pieces' fragments of four and the sums over small scale blocks would not fit the
 * registers), and the segments of K that blocks make of them, of as many waves as the kernels' registers allow: le_g4t_* 16 with one set, or
 * with two at scale blocks of 64 and more (16 / 8 waves, two tokens fp32 in groups of 64: 5120 x 5120, one segment against two, 9.4 /
 * 12.2 us, 4096 x 14336, two against four, 14.7 / 15.3, 28672 x 8192 32.2 / 32.2); 12 with two sets of two pieces at 32 or three at 64 and
 * more, where that makes one segment (12 / 8, five tokens: 5120 x 5120 12.3 / 15.1 us; but 4096 x 14336, three against four, 21.4 / 18.8);
 * else, and le_g4m_*, eight. */
int chunks(const le_g4 *w, int xtype, int swiglu, int m) { return !row_sets(xtype, swiglu, m) && pieces16(xtype, swiglu) == 2 && scale_block(w) == 32 ? 2 : 4; }
int segments(const le_g4 *w, int xtype, int swiglu, int m) {
    const int na = row_sets(xtype, swiglu, m), sub = scale_block(w), nc = (w->cols + 127) / 128;
    const bool w16 = na == 1 || (na == 2 && sub >= 64), w12 = (na == 3 && sub >= 64) || (na == 2 && pieces16(xtype, swiglu) == 2);
    const int most = (w16 ? 16 : w12 && nc <= 12 * 4 ? 12 : 8) * chunks(w, xtype, swiglu, m);
    return (nc + most - 1) / most;
}
/* What is wrong with a shape, or null. */
const char *shape_error(const le_g4 *w, int slots, int share, int m) {
    if (w->n_mat <= 0 || w->rows <= 0 || w->cols <= 0 || slots <= 0 || share <= 0 || m <= 0) return "empty shape";
    if (w->cols % 32) return "cols is not a multiple of 32";
    if (w->group != w->cols && (w->group < 32 || (w->group & (w->group - 1)) || w->cols % w->group))
        return "group is neither cols nor a power of two from 32 on that divides cols";
    if (m > 64 || slots > 65535 || w->cols > 1 << 24) return "m above 64, slots above 65535 or cols above 2^24";
    if ((long long)slots * m * w->rows > 1LL << 31) return "more than 2^31 results";
    if ((long long)w->rows * (w->cols / 2) >= 1LL << 32 || (long long)w->rows * (w->cols / w->group) * type_bytes(w->scale_type) >= 1LL << 32)
        return "a matrix with codes or scales of 4 GiB or more";
    return nullptr;
}

}  // namespace

extern "C" size_t le_matvec_g4_workspace_size(const le_g4 *w, int xtype, int m, int slots, int share, int swiglu) {
    if (!w || !type_bytes(xtype) || !type_bytes(w->scale_type) || shape_error(w, slots, share, m) || m <= most_tokens(xtype, swiglu)) return 0;
    const int segs = segments(w, xtype, swiglu, m);
    return (size_t)((slots + share - 1) / share) * set_bytes(xtype, swiglu, m, w->cols) + (segs > 1 ? (size_t)segs * slots * m * w->rows * 4 : 0);
}

extern "C" int le_matvec_g4(le_ctx *c, const le_g4 *w, const int *sel, int slots, int share, int xtype, const void *x,
                            long long xstride, int m, void *y, int swiglu, void *ws, size_t ws_bytes,
                            le_stream_t stream) {
    if (!c) return LE_ERR_ARG;
    if (!w || !w->codes || !w->scales || !x || !y) return le_ctx_fail(c, LE_ERR_ARG, "null pointer");
    const int xb = type_bytes(xtype), sb = type_bytes(w->scale_type);
    if (!xb) return le_ctx_failf(c, LE_ERR_TYPE, "activations of type %d", xtype);
    if (!sb) return le_ctx_failf(c, LE_ERR_TYPE, "scales of type %d", w->scale_type);
    if (const char *e = shape_error(w, slots, share, m))
        return le_ctx_failf(c, LE_ERR_SHAPE, "%s (%d matrices of %d x %d, group %d; %d slots, %d sharing, %d tokens)", e, w->n_mat, w->rows, w->cols, w->group, slots, share, m);
    if (!sel && slots > w->n_mat) return le_ctx_failf(c, LE_ERR_SHAPE, "%d slots of %d matrices without sel", slots, w->n_mat);
    const long long width = swiglu ? 2LL * w->cols : w->cols;
    if (xstride && xstride < width) return le_ctx_failf(c, LE_ERR_SHAPE, "xstride=%lld is less than a row of %lld", xstride, width);
    if (!aligned(w->codes, 16) || !aligned(x, 16) || xstride % (16 / xb))
        return le_ctx_fail(c, LE_ERR_ALIGN, "codes, x and its rows must be 16-byte aligned");
    if (!aligned(w->scales, sb) || !aligned(w->zeros, sb) || !aligned(y, xb) || !aligned(sel, 4))
        return le_ctx_fail(c, LE_ERR_ALIGN, "scales, zeros, sel and y must be aligned to their types");
    const size_t need = le_matvec_g4_workspace_size(w, xtype, m, slots, share, swiglu);
    if (need && (!ws || ws_bytes < need)) return le_ctx_failf(c, LE_ERR_WORKSPACE, "workspace needs %zu bytes", need);
    if (need && !aligned(ws, 16)) return le_ctx_fail(c, LE_ERR_ALIGN, "ws must be 16-byte aligned");
    if (need && (long long)((slots + share - 1) / share) * m > 65535) return le_ctx_fail(c, LE_ERR_SHAPE, "more than 65535 tokens");
    if (int rc = le_ctx_on_device(c)) return rc;
    G4Args a{};
    a.codes = (const unsigned char *)w->codes;
    a.scales = w->scales;
    a.zeros = w->zeros;
    a.sel = sel;
    a.x = x;
    a.y = y;
    a.xstride = xstride;
    a.n_mat = w->n_mat;
    a.rows = w->rows;
    a.cols = w->cols;
    a.group = w->group;
    a.ng = w->cols / w->group;
    a.share = share;
    a.m = m;
    a.gshift = 31; /* one group a row */
    if (w->group != w->cols)
        for (a.gshift = 5; 1 << a.gshift < w->group;) a.gshift++;
    a.xty = xtype;
    const int sub = scale_block(w), bpc = 128 / sub;
    /* a 128-column part's scales and its zero points can be loaded at once */
    const bool vec = bpc > 1 && a.ng % bpc == 0 && aligned(w->scales, bpc * sb) && aligned(w->zeros, bpc * sb);
    char tail[16];
    snprintf(tail, sizeof tail, "b%d%s", sub, vec ? "v" : "");
    const char *kind = xtype == LE_F32 ? "f32" : xtype == LE_F16 ? "f16" : "bf16";
    const long long groups = (w->rows + 15) / 16;
    const int most = most_tokens(xtype, swiglu), sty = w->scale_type, P = pieces(xtype, swiglu);
    char name[48];
    void *args[] = {&a};
    /* Row groups a block: so many that blocks of nw waves, for each of the `others` (slots, token tiles, segments), fill the chip with
     * `waves` a CU once or, where a block's LDS (lds bytes a wave and row group, `fixed` beside them) cannot hold its groups'
     * partial results then, R times; then the fewest blocks that need no more groups (14336 x 4096 fp32, four tokens: 224 blocks 12.8 us,
     * 256 with 3 or 4 groups 13.5). Rounds that end short are what this avoids: the same matrix with 64 tokens, in blocks of 8 groups
     * for 64 KB 41.8 us, now 34.7; 40 tokens in groups of 32 47.7, now 44.4; 32000 x 4096, 5 tokens 31.4, now 25.8 (bf16, whose kernel fits a CU
     * twice, 21.1, now 22.2). */
    auto share_out = [&](int nw, int waves, long long others, int lds, int fixed) {
        const int blocks = std::max(1, waves / nw); /* a CU */
        const long long target = (long long)le_ctx_cus(c) * blocks, cap = std::max(1, (144 * 1024 / blocks - fixed) / (nw * lds));
        const long long least = (groups + cap - 1) / cap, R = (least * others + target - 1) / target;
        const long long most_gx = std::min(groups, target * R / others), per = (groups + most_gx - 1) / most_gx, gx = (groups + per - 1) / per;
        a.nw = nw;
        a.gx = (int)gx;
        a.per = (int)per;
        a.full = (int)(groups - (a.per - 1) * gx);
    };
    if (m <= most) {
        /* slices of 512 columns; 16 waves a block for more than eight of them (but for several tokens at scale blocks of 32, which take
         * more than the 128 registers that leaves): 4096 x 14336 in groups of 64, 16 / 8 waves, fp32 11.3 / 12.3 us, SwiGLU 13.0 /
         * 13.7, bf16, 4 tokens 14.6 / 15.1; 2048 x 6144 SwiGLU 6.75 / 7.8 */
        const int ns = (w->cols + 511) / 512, wmax = ns <= 8 || (sub < 64 && m > 1) ? 8 : 16;
        const int passes = (ns + wmax - 1) / wmax, nw = (ns + passes - 1) / passes, T = m == 1 ? 1 : most;
        const int quad = m == 1 && P > 1 ? nw * 4096 : 0;
        /* 32 experts of 1536 x 2048 (four waves a block), 16 / 24 waves a CU: groups of 32 15.0 / 14.4 us, 128 12.1 / 11.7; 28672 x
         * 4096 (eight) 13.1 / 14.6 */
        share_out(nw, nw <= 4 ? 24 : 16, slots, T * 256, quad);
        snprintf(name, sizeof name, "le_g4q_%s%s_%s%s_s%d", kind, swiglu ? "w" : m == 1 ? "" : T == 2 ? "t2" : "t4", tail, passes > 1 || nw > 8 ? "_mp" : "", sty);
        return le_ctx_launch(c, name, dim3((unsigned)a.gx, (unsigned)slots), 64 * nw, (size_t)quad + (size_t)a.per * nw * T * 256, (hipStream_t)stream, args);
    }
    a.ws = (unsigned char *)ws;
    a.ws_set = (long long)set_bytes(xtype, swiglu, m, w->cols);
    a.ws_downs = (long long)frag_bytes(xtype, swiglu, m, w->cols);
    a.na = row_sets(xtype, swiglu, m);
    a.segs = segments(w, xtype, swiglu, m);
    const int sets = (slots + share - 1) / share, nc = (w->cols + 127) / 128, tiles = a.na ? 1 : (m + 15) / 16, cs = chunks(w, xtype, swiglu, m);
    a.part = (float *)(a.ws + sets * a.ws_set);
    a.total = (long long)slots * m * w->rows;
    snprintf(name, sizeof name, "le_g4x_%s%s_b%d", kind, swiglu ? "w" : "", sub);
    int rc = le_ctx_launch(c, name, dim3((unsigned)((nc * 16 + 255) / 256), (unsigned)(sets * m)), 256, 0, (hipStream_t)stream, args);
    if (rc) return rc;
    /* waves: all of K's slices over the segments, evenly */
    const int nw = ((nc + cs - 1) / cs + a.segs - 1) / a.segs, p16 = pieces16(xtype, swiglu), lds = a.na ? a.na * 4 / p16 * 256 : 1024;
    share_out(nw, 8, (long long)slots * tiles * a.segs, lds, 0);
    if (a.na) snprintf(name, sizeof name, "le_g4t_n%d_p%d_%s%s_s%d", a.na, p16, tail, nw > 8 && a.na == 2 && p16 == 1 && sub == 64 ? "_w" : "", sty);
    else snprintf(name, sizeof name, "le_g4m_p%d_%s_s%d", p16, tail, sty);
    rc = le_ctx_launch(c, name, dim3((unsigned)a.gx, (unsigned)slots, (unsigned)(tiles * a.segs)), 64 * nw, (size_t)a.per * nw * lds, (hipStream_t)stream, args);
    if (rc || a.segs == 1) return rc;
    return le_ctx_launch(c, "le_g4s", dim3((unsigned)((a.total + 255) / 256)), 256, 0, (hipStream_t)stream, args);
}
