/* Host side of the routed experts' products (le_mm_experts and its gradients, include/le_qmm.h): argument checks and launch shapes. */
#include <algorithm>
#include <cstdio>

#include "le_checks.h"
#include "le_ctx.h"
#include "le_experts_args.h"

namespace {

constexpr int kSide = 1 << 24, kExperts = 1024, kRows = 1 << 30, kCus = 256;

bool size_error(int n_exp, int n_row, int rows, int cols) {
    return n_exp <= 0 || n_exp > kExperts || n_row < 0 || n_row > kRows || rows <= 0 || cols <= 0 || rows > kSide || cols > kSide;
}

int check_sizes(le_ctx *c, int ty, int n_exp, int n_row, int rows, int cols, long long ldx, long long ldy) {
    if (!le_type_bytes(ty)) return le_ctx_failf(c, LE_ERR_TYPE, "rows of type %d", ty);
    if (size_error(n_exp, n_row, rows, cols))
        return le_ctx_failf(c, LE_ERR_SHAPE, "n_exp=%d (1..1024), n_row=%d (0..2^30), rows=%d, cols=%d (1..2^24)", n_exp, n_row, rows, cols);
    if (ldx < cols || ldy < rows) return le_ctx_failf(c, LE_ERR_SHAPE, "row strides %lld and %lld of %d and %d values", ldx, ldy, cols, rows);
    return LE_OK;
}

/* Into how many parts the weights' gradient cuts an expert's rows, each with sums of its own in the workspace: two blocks a CU where there are
 * fewer tiles of 128 x 128 than CUs, of 256 rows and more on average. */
int parts(int n_exp, int n_row, int rows, int cols) {
    const long long tiles = ((rows + 127LL) / 128) * ((cols + 127LL) / 128) * n_exp;
    if (tiles >= kCus) return 1;
    return (int)std::max(1LL, std::min({2 * kCus / tiles, n_row / (256LL * n_exp), 64LL}));
}

/* Whether y is taken by a wave a tile: few rows an expert, fewer where a wave's work on them is short (us, so / in larger tiles, 128 experts bf16:
 * 1536 x 2048 64 rows 60 / 65, 256 rows 110 / 119, 512 rows 130 / 127; 2048 x 768 64 rows 33 / 37, 128 rows 58 / 54; 8 of 14336 x 4096 16 rows
 * 150 / 189); fp32, bound by the matrix instructions, where larger tiles are fewer than CUs (8 rows 43 / 88, 64 rows 209 / 145). */
bool few_rows(const ExpertArgs &a, int ty, const char *what) {
    if (what[0] != 'y' || a.n_row >= (a.k * (long long)le_type_bytes(ty) < 4096 ? 1LL : 3LL) * a.n_exp) return false;
    return ty != LE_F32 || std::min(a.n_exp, a.n_row) * ((a.n + 255LL) / 256) < kCus;
}

/* The kernel of `what`_type. whole: every row that is read is whole 16-byte chunks. */
int launch(le_ctx *c, const char *what, int ty, ExpertArgs &a, bool whole, le_stream_t stream) {
    const bool dw = what[1] == 'w';
    int bm = 128, bn = 128;
    /* tiles of 128 x 128 and of 128 x 256 that there may be (times below: of this choice / of the other) */
    const bool f32 = ty == LE_F32;
    const long long row_tiles = a.n_row / 128 + std::min(a.n_exp, a.n_row), t128 = row_tiles * ((a.n + 127LL) / 128), t256 = row_tiles * ((a.n + 255LL) / 256);
    if (!dw && (whole ? f32 && t128 <= 512 && !few_rows(a, ty, what) : a.n_row < 48LL * a.n_exp || t128 < 256 || (f32 && t128 < 2048))) {
        /* tiles of 32 rows through registers for few rows an expert, or where larger tiles are too few (256 rows of 4 experts of 4096 x 4096
         * bf16 43 / 56 us); fp32 is bound by the matrix instructions, which more waves keep busier (1351 rows of 7 experts of 1951 x 1024:
         * dx 90 / 156, of 1952 x 1024 73 / 81; 16384 rows of 16 of 2048 x 1024 720 / 654) */
        bm = 32;
        whole = false;
    } else if (!whole) {
        if (dw && a.m <= 32) bm = 32;
    } else if (few_rows(a, ty, what)) {
        bm = bn = 32;
    } else if (dw) {
        /* a block a CU takes tile after tile of 256 x 256: not where CUs would stand idle for more than a fifth of the time (16384 rows of 8
         * experts of 1024 x 1024 bf16 69 / 47 us, 8192 of one of 4096 x 4096 264 / 310) */
        const long long wide = (a.m + 255LL) / 256 * ((a.n + 255LL) / 256) * a.n_exp, turns = (wide + kCus - 1) / kCus;
        if (a.n > 128 && 5 * wide >= 4 * turns * kCus) bm = bn = 256;
    } else if (!f32 && a.n > 128 && t256 >= 512) {
        /* two blocks a CU (16384 rows of 8 experts of 1024 x 1024 bf16 45 / 63 us, 8192 39 / 38, 2048 23 / 17); not fp32 (32768 rows of 128 of
         * 1536 x 2048 2198 / 2105) */
        bn = 256;
    }
    const bool few = bn == 32;
    int waves = 4;
    if (few) {
        /* waves by how many tiles there may be: four a tile (16 rows of one expert of 4096 x 4096 bf16 11 us, by one wave 21), or one (384 tiles: 14, by
         * four 20); more than the 1024 that run at once one after the other, so that none begins late (64 rows of 128 experts, of 2048 x 768
         * 33 / 42 us, of 1536 x 2048 60 / 62) */
        const long long most = (long long)std::min(a.n_exp, a.n_row) * ((a.n + 31LL) / 32);
        if (most > 256) waves = 1;
        if (a.n_row < 2LL * a.n_exp) a.strip = (int)std::max(1LL, std::min(most / 1024, 4LL));
        bn = 32 * a.strip;
    }
    a.mt = (a.m + bm - 1) / bm;
    a.nt = (a.n + bn - 1) / bn;
    const long long tiles = (dw ? (long long)a.mt * a.n_exp * a.segs : a.n_row / bm + std::min(a.n_exp, a.n_row)) * a.nt;
    if (tiles > 0x7FFFFFFFLL) return le_ctx_fail(c, LE_ERR_SHAPE, "more than 2^31 tiles");
    char name[40];
    if (few) snprintf(name, sizeof name, "le_ex_y_%d_few", ty);
    else if (whole) snprintf(name, sizeof name, "le_ex_%s_%d_m%d_n%d", what, ty, bm, bn);
    else snprintf(name, sizeof name, "le_ex_%s_%d_any%d", what, ty, bm);
    void *args[] = {&a};
    if (bm == 256) {
        /* a block a CU; the ring (three steps for fp32 results, whose rows take more of LDS, else four), the results of eight waves, off */
        const bool wide32 = f32 || what[2] == 'f';
        const size_t lds = (size_t)(wide32 ? 3 : 4) * 512 * 64 + 8 * 16 * (64 * (wide32 ? 4 : 2) + 16) + (size_t)(a.n_exp + 1) * 4;
        const int cus = std::max(8, le_ctx_cus(c));
        for (a.run = 1; a.run * 2 <= tiles / 8 && cus / 8 % (a.run * 2) == 0;) a.run *= 2;
        return le_ctx_launch(c, name, dim3((unsigned)(cus / (8 * a.run) * (8 * a.run))), 512, lds, (hipStream_t)stream, args);
    }
    /* tiles in whole turns of the eight XCDs, `run` in a row to each: an expert's, which share weights (18 in a row 351 us, 4 373, single ones 414) */
    a.run = (int)std::max(1LL, std::min({tiles / (a.n_exp * (long long)a.segs), tiles / 64, 1LL << 16}));
    const long long turn = 8LL * a.run;
    return le_ctx_launch(c, name, dim3((unsigned)std::min((tiles + turn - 1) / turn * turn, (1LL << 23) / turn * turn)), 64 * waves, few ? waves * 40960 : whole ? 3 * (bm + bn) * 64 : 0,
                         (hipStream_t)stream, args);
}
/* Whether rows of `rows` and `cols` values, ld1 and ld2 apart, are whole 16-byte chunks. */
bool whole_rows(int ty, const void *p, const void *q, long long ld1, long long ld2, int rows, int cols) {
    const int n = 16 / le_type_bytes(ty);
    return le_aligned(p, 16) && le_aligned(q, 16) && ld1 % n == 0 && ld2 % n == 0 && rows % n == 0 && cols % n == 0;
}

}  // namespace

extern "C" {

int le_mm_experts(le_ctx *c, int ty, const void *w, const int *off, int n_exp, const void *x, long long ldx, void *y,
                  long long ldy, int n_row, int rows, int cols, le_stream_t stream) {
    if (!c) return LE_ERR_ARG;
    if (int rc = check_sizes(c, ty, n_exp, n_row, rows, cols, ldx, ldy)) return rc;
    if (n_row == 0) return LE_OK;
    if (!w || !off || !x || !y) return le_ctx_fail(c, LE_ERR_ARG, "null pointer");
    const int b = le_type_bytes(ty);
    if (!le_aligned(w, b) || !le_aligned(x, b) || !le_aligned(y, b) || !le_aligned(off, 4))
        return le_ctx_fail(c, LE_ERR_ALIGN, "pointers must be aligned to their types");
    if (int rc = le_ctx_on_device(c)) return rc;
    ExpertArgs a{x, w, y, off, ldx, cols, ldy, n_exp, n_row, n_row, rows, cols, 0, 0, 1, 1, 1};
    return launch(c, "y", ty, a, whole_rows(ty, x, w, ldx, 0, cols, cols), stream);
}

int le_mm_experts_dx(le_ctx *c, int ty, const void *w, const int *off, int n_exp, const void *dy, long long ldy, void *dx,
                     long long ldx, int n_row, int rows, int cols, le_stream_t stream) {
    if (!c) return LE_ERR_ARG;
    if (int rc = check_sizes(c, ty, n_exp, n_row, rows, cols, ldx, ldy)) return rc;
    if (n_row == 0) return LE_OK;
    if (!w || !off || !dy || !dx) return le_ctx_fail(c, LE_ERR_ARG, "null pointer");
    const int b = le_type_bytes(ty);
    if (!le_aligned(w, b) || !le_aligned(dy, b) || !le_aligned(dx, b) || !le_aligned(off, 4))
        return le_ctx_fail(c, LE_ERR_ALIGN, "pointers must be aligned to their types");
    if (int rc = le_ctx_on_device(c)) return rc;
    ExpertArgs a{dy, w, dx, off, ldy, cols, ldx, n_exp, n_row, n_row, cols, rows, 0, 0, 1, 1, 1};
    return launch(c, "dx", ty, a, whole_rows(ty, dy, w, ldy, 0, rows, cols), stream);
}

size_t le_mm_experts_dw_workspace_size(int ty, int n_exp, int n_row, int rows, int cols) {
    if (!le_type_bytes(ty) || size_error(n_exp, n_row, rows, cols)) return 0;
    const int n = parts(n_exp, n_row, rows, cols);
    return n > 1 ? (size_t)n * n_exp * rows * cols * 4 : 0;
}

int le_mm_experts_dw(le_ctx *c, int ty, const void *dy, long long ldy, const void *x, long long ldx, const int *off, int n_exp,
                     int dwtype, void *dw, int n_row, int rows, int cols, void *ws, size_t ws_bytes, le_stream_t stream) {
    if (!c) return LE_ERR_ARG;
    if (int rc = check_sizes(c, ty, n_exp, n_row, rows, cols, ldx, ldy)) return rc;
    if (dwtype != ty && dwtype != LE_F32) return le_ctx_failf(c, LE_ERR_TYPE, "dw of type %d for rows of type %d", dwtype, ty);
    if (!off || !dw || (n_row && (!dy || !x))) return le_ctx_fail(c, LE_ERR_ARG, "null pointer");
    const int b = le_type_bytes(ty);
    if (!le_aligned(dy, b) || !le_aligned(x, b) || !le_aligned(dw, le_type_bytes(dwtype)) || !le_aligned(off, 4) || !le_aligned(ws, 16))
        return le_ctx_fail(c, LE_ERR_ALIGN, "pointers must be aligned to their types, ws to 16 bytes");
    const size_t need = le_mm_experts_dw_workspace_size(ty, n_exp, n_row, rows, cols);
    if (need && (!ws || ws_bytes < need)) return le_ctx_failf(c, LE_ERR_WORKSPACE, "workspace needs %zu bytes", need);
    ExpertArgs a{dy, x, dw, off, ldy, ldx, cols, n_exp, n_row, rows, cols, n_row, 0, 0, 1, parts(n_exp, n_row, rows, cols), 1};
    if (int rc = le_ctx_on_device(c)) return rc;
    const bool whole = whole_rows(ty, dy, x, ldy, ldx, rows, cols);
    const char *what = dwtype == ty ? "dw" : "dwf";
    if (a.segs == 1) return launch(c, what, ty, a, whole, stream);
    a.y = ws;
    if (int rc = launch(c, ty == LE_F32 ? "dw" : "dwf", ty, a, whole, stream)) return rc;
    char name[40];
    snprintf(name, sizeof name, "le_ex_%s_%d_sum", what, ty);
    int n = n_exp * rows * cols; /* at most 2^22, since there are fewer than 256 tiles */
    void *args[] = {&ws, &dw, &n, &a.segs};
    return le_ctx_launch(c, name, dim3((unsigned)((n + 255) / 256)), 256, 0, (hipStream_t)stream, args);
}

}  // extern "C"
