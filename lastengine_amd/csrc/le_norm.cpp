/* Host side of le_add_rms_quant (include/le_qmm.h): argument checks and launch shape. */
#include <algorithm>
#include <cmath>
#include <cstdio>

#include "le_checks.h"
#include "le_ctx.h"
#include "le_norm_args.h"

extern "C" int le_add_rms_quant(le_ctx *c, int ty, const void *x, long long ldx, const void *res, long long ldr, const float *w, void *h,
                                long long ldh, void *o, long long ldo, int8_t *xq, float *xd, int32_t *xs, int m, int n, float eps,
                                le_stream_t stream) {
    if (!c) return LE_ERR_ARG;
    const int b = le_type_bytes(ty);
    if (!b) return le_ctx_failf(c, LE_ERR_TYPE, "rows of type %d", ty);
    if (m < 0 || n <= 0 || n > 1 << 24 || (xq && n % 32)) return le_ctx_failf(c, LE_ERR_SHAPE, "m=%d, n=%d (1..2^24, with xq a multiple of 32)", m, n);
    if (ldx < n || (res && ldr < n) || (h && ldh < n) || (o && ldo < n))
        return le_ctx_failf(c, LE_ERR_SHAPE, "row strides %lld, %lld, %lld and %lld of %d values", ldx, ldr, ldh, ldo, n);
    if (!(eps >= 0.f) || std::isinf(eps)) return le_ctx_failf(c, LE_ERR_ARG, "eps=%g", eps);
    if (!xq != !xd || (xs && !xq)) return le_ctx_fail(c, LE_ERR_ARG, "xq and xd go together, and xs with them");
    if (m == 0) return LE_OK;
    if (!x || !w || (!h && !o && !xq)) return le_ctx_fail(c, LE_ERR_ARG, "null pointer");
    if ((h == x && ldh != ldx) || (h && h == res && ldh != ldr)) return le_ctx_fail(c, LE_ERR_ARG, "h in place of x or res has its row stride");
    if (!le_aligned(x, b) || !le_aligned(res, b) || !le_aligned(h, b) || !le_aligned(o, b) || !le_aligned(w, 4) || !le_aligned(xd, 4) || !le_aligned(xs, 4))
        return le_ctx_fail(c, LE_ERR_ALIGN, "pointers must be aligned to their types");
    if (int rc = le_ctx_on_device(c)) return rc;
    NormArgs a{x, res, w, h, o, (signed char *)xq, xd, xs, ldx, ldr, ldh, ldo, m, n, eps};
    void *args[] = {&a};
    const int V = 16 / b, pieces = (n + V - 1) / V;
    char name[40];
    if (n % V || pieces > 4096) {
        const int L = pieces <= 1024 ? 256 : 1024;
        snprintf(name, sizeof name, "le_nq_%d_any%d", ty, L);
        return le_ctx_launch(c, name, dim3((unsigned)std::min(m, 1 << 20)), L, 0, (hipStream_t)stream, args);
    }
    /* lanes a row: a wave up to 128 pieces; from there a block of 256 (64 / 256 lanes: 1024 rows of 2048 bf16 9.5 / 7.0 us, 4096 rows 21 / 17, 2048
     * rows of 1024 fp32 9.5 / 8.3), beyond 1024 pieces one of 1024; four times as many while the rows do not fill the chip (256 / 1024: 8 rows
     * of 4096 fp32 5.9 / 5.1 us, 256 rows 7.3 / 6.6, 1024 rows 14.0 / 15.6) */
    int L = pieces <= 128 ? 64 : pieces <= 1024 ? 256 : 1024, nc = 1;
    while (L < 1024 && pieces > L && (long long)m * L <= 256LL * le_ctx_cus(c)) L *= 4;
    while (nc * L < pieces) nc *= 2;
    snprintf(name, sizeof name, "le_nq_%d_l%d_c%d", ty, L, nc);
    return le_ctx_launch(c, name, dim3((unsigned)std::min(L == 64 ? (m + 3LL) / 4 : m, 1LL << 20)), L == 64 ? 256 : L, 0, (hipStream_t)stream, args);
}
