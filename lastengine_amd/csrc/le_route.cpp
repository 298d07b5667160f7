/* Host side of the expert-routing entries (le_moe_route, le_moe_sort, le_moe_permute, le_moe_combine and their gradients,
 * include/le_qmm.h): argument checks and launch shapes. */
#include <algorithm>
#include <cstdint>
#include <cstdio>
#include <cstring>

#include "le_ctx.h"
#include "le_route_args.h"

namespace {

int type_bytes(int ty) { return ty == LE_F32 ? 4 : ty == LE_F16 || ty == LE_BF16 ? 2 : 0; }
bool aligned(const void *p, unsigned n) { return ((uintptr_t)p & (n - 1)) == 0; }

/* The counts every entry takes. */
int check_pairs(le_ctx *c, int n_tok, int k) {
    if (n_tok < 0 || k <= 0 || k > 16 || (long long)n_tok * k > 0x7FFFFFFFLL)
        return le_ctx_failf(c, LE_ERR_SHAPE, "n_tok=%d, k=%d: k is 1..16 and there are fewer than 2^31 pairs", n_tok, k);
    return LE_OK;
}
int check_experts(le_ctx *c, int n_exp, int k_most) {
    if (n_exp <= 0 || n_exp > 1024 || k_most > n_exp)
        return le_ctx_failf(c, LE_ERR_SHAPE, "n_exp=%d (1..1024) or k above it", n_exp);
    return LE_OK;
}
int check_rows(le_ctx *c, int ty, long long ldt, long long lde, int n_tok, int k, int cols, int n_row) {
    if (!type_bytes(ty)) return le_ctx_failf(c, LE_ERR_TYPE, "rows of type %d", ty);
    if (int rc = check_pairs(c, n_tok, k)) return rc;
    if (cols <= 0 || cols > 1 << 25 || n_row < 0 || ldt < cols || lde < cols)
        return le_ctx_failf(c, LE_ERR_SHAPE, "cols=%d (1..2^25), n_row=%d, row strides %lld and %lld", cols, n_row, ldt, lde);
    return LE_OK;
}

/* How le_rt_sort takes np pairs: one block up to 4096 of them, else at most 256 blocks of 16 waves. */
struct SortShape {
    int blocks = 1, waves, steps;
    explicit SortShape(int np) {
        waves = std::max(1, (int)std::min(16LL, (np + 63LL) / 64));
        const int one = (int)((np + 1023LL) / 1024); /* steps of one block */
        steps = std::max(1, one);
        if (np > 4096) {
            steps = (one + 255) / 256;
            blocks = (int)((np + 1024LL * steps - 1) / (1024LL * steps));
        }
    }
};

}  // namespace

extern "C" {

int le_moe_route(le_ctx *c, int ltype, const void *logits, int n_tok, int n_exp, int k, int *idx, float *w,
                 le_stream_t stream) {
    if (!c) return LE_ERR_ARG;
    const int b = type_bytes(ltype);
    if (!b) return le_ctx_failf(c, LE_ERR_TYPE, "logits of type %d", ltype);
    if (int rc = check_pairs(c, n_tok, k)) return rc;
    if (int rc = check_experts(c, n_exp, k)) return rc;
    if (n_tok == 0) return LE_OK;
    if (!logits || !idx || !w) return le_ctx_fail(c, LE_ERR_ARG, "null pointer");
    if (!aligned(logits, b) || !aligned(idx, 4) || !aligned(w, 4)) return le_ctx_fail(c, LE_ERR_ALIGN, "pointers must be aligned to their types");
    if (int rc = le_ctx_on_device(c)) return rc;
    RouteArgs a{logits, idx, w, n_tok, n_exp, k};
    void *args[] = {&a};
    /* lanes a token and experts a lane: 64 lanes while the waves do not fill the chip (and for many experts), else the fewest
     * that hold the experts in eight values each */
    int L = n_exp <= 128 ? 16 : n_exp <= 256 ? 32 : 64, V = n_exp <= 32 ? 2 : n_exp <= 64 ? 4 : n_exp <= 512 ? 8 : 16;
    if (L < 64 && n_tok <= 8 * le_ctx_cus(c)) L = 64, V = n_exp <= 64 ? 1 : n_exp <= 128 ? 2 : 4;
    char name[40];
    snprintf(name, sizeof name, "le_rt_route_%d_l%d_v%d", ltype, L, V);
    return le_ctx_launch(c, name, dim3((unsigned)std::min((n_tok * (long long)L + 255) / 256, 1LL << 20)), 256, 0, (hipStream_t)stream, args);
}

int le_moe_route_bwd(le_ctx *c, int ltype, const int *idx, const float *w, const float *dw, int n_tok, int n_exp, int k,
                     void *dlogits, le_stream_t stream) {
    if (!c) return LE_ERR_ARG;
    const int b = type_bytes(ltype);
    if (!b) return le_ctx_failf(c, LE_ERR_TYPE, "logits of type %d", ltype);
    if (int rc = check_pairs(c, n_tok, k)) return rc;
    if (int rc = check_experts(c, n_exp, k)) return rc;
    if (n_tok == 0) return LE_OK;
    if (!idx || !w || !dw || !dlogits) return le_ctx_fail(c, LE_ERR_ARG, "null pointer");
    if (!aligned(dlogits, b) || !aligned(idx, 4) || !aligned(w, 4) || !aligned(dw, 4))
        return le_ctx_fail(c, LE_ERR_ALIGN, "pointers must be aligned to their types");
    if (int rc = le_ctx_on_device(c)) return rc;
    RouteBwdArgs a{idx, w, dw, dlogits, n_tok, n_exp, k};
    void *args[] = {&a};
    char name[32];
    snprintf(name, sizeof name, "le_rt_route_bwd_%d", ltype);
    return le_ctx_launch(c, name, dim3((unsigned)std::min((n_tok + 3LL) / 4, 1LL << 20)), 256, 0, (hipStream_t)stream, args);
}

size_t le_moe_sort_workspace_size(int n_tok, int k, int n_exp) {
    if (n_tok < 0 || k <= 0 || k > 16 || (long long)n_tok * k > 0x7FFFFFFFLL || n_exp <= 0 || n_exp > 1024) return 0;
    const SortShape s(n_tok * k);
    return s.blocks > 1 ? (size_t)s.blocks * n_exp * 4 : 0;
}

int le_moe_sort(le_ctx *c, const int *idx, int n_tok, int k, int n_exp, int *off, int *in_idx, int *out_idx, int *pos,
                void *ws, size_t ws_bytes, le_stream_t stream) {
    if (!c) return LE_ERR_ARG;
    if (int rc = check_pairs(c, n_tok, k)) return rc;
    if (int rc = check_experts(c, n_exp, 0)) return rc;
    if (!off || (!idx && n_tok)) return le_ctx_fail(c, LE_ERR_ARG, "null pointer");
    if (!aligned(idx, 4) || !aligned(off, 4) || !aligned(in_idx, 4) || !aligned(out_idx, 4) || !aligned(pos, 4) || !aligned(ws, 16))
        return le_ctx_fail(c, LE_ERR_ALIGN, "pointers must be aligned to their types, ws to 16 bytes");
    const size_t need = le_moe_sort_workspace_size(n_tok, k, n_exp);
    if (need && (!ws || ws_bytes < need)) return le_ctx_failf(c, LE_ERR_WORKSPACE, "workspace needs %zu bytes", need);
    if (int rc = le_ctx_on_device(c)) return rc;
    const SortShape s(n_tok * k);
    SortArgs a{idx, off, in_idx, out_idx, pos, n_tok * k, k, n_exp, s.blocks, s.waves, s.steps, (int *)ws};
    void *args[] = {&a};
    if (s.blocks > 1)
        if (int rc = le_ctx_launch(c, "le_rt_count", dim3((unsigned)s.blocks), 64 * s.waves, (size_t)n_exp * 4, (hipStream_t)stream, args)) return rc;
    return le_ctx_launch(c, "le_rt_sort", dim3((unsigned)s.blocks), 64 * s.waves, ((size_t)(s.waves + 2) * n_exp + 16) * 4, (hipStream_t)stream, args);
}

static int rows_launch(le_ctx *c, const char *what, int ty, const RowsArgs &rows, le_stream_t stream) {
    if (int rc = le_ctx_on_device(c)) return rc;
    RowsArgs a = rows;
    void *args[] = {&a};
    /* lanes a token: as many as its row has 16-byte parts, of 16, 64 and 256; longer rows are cut over the grid's second axis where
     * nothing is summed over a row */
    const int n = ty == LE_F32 ? 4 : 8, parts = (a.cols + n - 1) / n, L = parts <= 16 ? 16 : parts <= 64 ? 64 : 256;
    const bool whole = !strcmp(what, "combine_bwd");
    char name[40];
    /* expert rows that are read and lie at 16-byte addresses: non-temporal from 8 MB on (4096 tokens of 8 pairs by 2048 bf16: sum 30.3 -> 26.6
     * us, its gradient 62 -> 58, a sum behind that 90 -> 80; 64 tokens 3.6 -> 4.0, 301 by 1001 fp32, whose rows share lines, 5.3 -> 6.4) */
    const void *e = whole ? a.e : a.src;
    const int b = type_bytes(ty);
    const bool nt = strcmp(what, "permute") && e && (long long)a.n_tok * a.k * a.cols * b >= 8 << 20 && aligned(e, 16) && a.lde * b % 16 == 0;
    snprintf(name, sizeof name, "le_rt_%s_%d_l%d%s", what, ty, L, nt ? "_nt" : "");
    return le_ctx_launch(c, name, dim3((unsigned)std::min((a.n_tok * (long long)L + 255) / 256, 1LL << 20), whole ? 1u : (unsigned)((parts + L - 1) / L)), 256, 0,
                         (hipStream_t)stream, args);
}

int le_moe_permute(le_ctx *c, int ty, const void *x, long long ldt, const int *pos, int n_tok, int k, int cols, void *e,
                   long long lde, int n_row, le_stream_t stream) {
    if (!c) return LE_ERR_ARG;
    if (int rc = check_rows(c, ty, ldt, lde, n_tok, k, cols, n_row)) return rc;
    if (n_tok == 0 || n_row == 0) return LE_OK;
    if (!x || !e) return le_ctx_fail(c, LE_ERR_ARG, "null pointer");
    if (!aligned(x, type_bytes(ty)) || !aligned(e, type_bytes(ty)) || !aligned(pos, 4))
        return le_ctx_fail(c, LE_ERR_ALIGN, "pointers must be aligned to their types");
    return rows_launch(c, "permute", ty, RowsArgs{x, nullptr, e, pos, nullptr, nullptr, ldt, lde, n_tok, k, cols, n_row}, stream);
}

int le_moe_combine(le_ctx *c, int ty, const void *e, long long lde, int n_row, const int *pos, const float *w, int n_tok,
                   int k, int cols, void *out, long long ldt, le_stream_t stream) {
    if (!c) return LE_ERR_ARG;
    if (int rc = check_rows(c, ty, ldt, lde, n_tok, k, cols, n_row)) return rc;
    if (n_tok == 0) return LE_OK;
    if (!out || (!e && n_row)) return le_ctx_fail(c, LE_ERR_ARG, "null pointer");
    if (!aligned(e, type_bytes(ty)) || !aligned(out, type_bytes(ty)) || !aligned(pos, 4) || !aligned(w, 4))
        return le_ctx_fail(c, LE_ERR_ALIGN, "pointers must be aligned to their types");
    return rows_launch(c, "combine", ty, RowsArgs{e, nullptr, out, pos, w, nullptr, ldt, lde, n_tok, k, cols, n_row}, stream);
}

int le_moe_combine_bwd(le_ctx *c, int ty, const void *dout, long long ldt, const void *e, long long lde, int n_row,
                       const int *pos, const float *w, int n_tok, int k, int cols, void *de, float *dw, le_stream_t stream) {
    if (!c) return LE_ERR_ARG;
    if (int rc = check_rows(c, ty, ldt, lde, n_tok, k, cols, n_row)) return rc;
    if (n_tok == 0 || (!de && !dw)) return LE_OK;
    if (!dout || (dw && !e && n_row)) return le_ctx_fail(c, LE_ERR_ARG, "null pointer");
    const int b = type_bytes(ty);
    if (!aligned(dout, b) || !aligned(e, b) || !aligned(de, b) || !aligned(pos, 4) || !aligned(w, 4) || !aligned(dw, 4))
        return le_ctx_fail(c, LE_ERR_ALIGN, "pointers must be aligned to their types");
    return rows_launch(c, "combine_bwd", ty, RowsArgs{dout, e, de, pos, w, dw, ldt, lde, n_tok, k, cols, n_row}, stream);
}

}  // extern "C"
