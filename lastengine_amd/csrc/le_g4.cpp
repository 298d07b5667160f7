/* Host side of the matrix-vector products with 4-bit codes and group scales (le_matvec_g4, include/le_qmm.h): argument
 * checks and launch shapes. */
#include <cstdint>
#include <cstdio>

#include "le_ctx.h"
#include "le_g4_args.h"

namespace {

int type_bytes(int ty) { return ty == LE_F32 ? 4 : ty == LE_F16 || ty == LE_BF16 ? 2 : 0; }
bool aligned(const void *p, unsigned n) { return ((uintptr_t)p & (n - 1)) == 0; }

}  // namespace

extern "C" int le_matvec_g4(le_ctx *c, const le_g4 *w, const int *sel, int slots, int share, int xtype, const void *x,
                            long long xstride, int m, void *y, int swiglu, le_stream_t stream) {
    if (!c) return LE_ERR_ARG;
    if (!w || !w->codes || !w->scales || !x || !y) return le_ctx_fail(c, LE_ERR_ARG, "null pointer");
    const int xb = type_bytes(xtype), sb = type_bytes(w->scale_type);
    if (!xb) return le_ctx_failf(c, LE_ERR_TYPE, "activations of type %d", xtype);
    if (!sb) return le_ctx_failf(c, LE_ERR_TYPE, "scales of type %d", w->scale_type);
    if (w->n_mat <= 0 || w->rows <= 0 || w->cols <= 0 || slots <= 0 || share <= 0 || m <= 0)
        return le_ctx_fail(c, LE_ERR_SHAPE, "empty shape");
    if (w->cols % 32) return le_ctx_failf(c, LE_ERR_SHAPE, "cols=%d is not a multiple of 32", w->cols);
    if (w->group != w->cols && (w->group < 32 || (w->group & (w->group - 1)) || w->cols % w->group))
        return le_ctx_failf(c, LE_ERR_SHAPE, "group=%d is neither cols nor a power of two from 32 on that divides cols=%d", w->group, w->cols);
    if (m > 64 || slots > 65535) return le_ctx_failf(c, LE_ERR_SHAPE, "m=%d above 64 or slots=%d above 65535", m, slots);
    if (w->rows > 1 << 27) return le_ctx_failf(c, LE_ERR_SHAPE, "rows=%d above 2^27", w->rows);
    if (!sel && slots > w->n_mat) return le_ctx_failf(c, LE_ERR_SHAPE, "%d slots of %d matrices without sel", slots, w->n_mat);
    const long long width = swiglu ? 2LL * w->cols : w->cols;
    if (xstride && xstride < width) return le_ctx_failf(c, LE_ERR_SHAPE, "xstride=%lld is less than a row of %lld", xstride, width);
    if (!aligned(w->codes, 16) || !aligned(x, 16) || xstride % (16 / xb))
        return le_ctx_fail(c, LE_ERR_ALIGN, "codes, x and its rows must be 16-byte aligned");
    if (!aligned(w->scales, sb) || !aligned(w->zeros, sb) || !aligned(y, xb) || !aligned(sel, 4))
        return le_ctx_fail(c, LE_ERR_ALIGN, "scales, zeros, sel and y must be aligned to their types");
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
    char name[48];
    snprintf(name, sizeof name, "le_g4_x%d_s%d_%s", xtype, w->scale_type, swiglu ? "swiglu" : "plain");
    void *args[] = {&a};
    return le_ctx_launch(c, name, dim3((unsigned)((w->rows + 15) / 16), (unsigned)slots, (unsigned)m), 256, 0,
                         (hipStream_t)stream, args);
}
