/* Host side of the low-rank adapters (le_lora, include/le_qmm.h): argument checks and launch shapes. */
#include <algorithm>
#include <cstdio>

#include "le_checks.h"
#include "le_ctx.h"
#include "le_lora_args.h"

namespace {

constexpr int kFew = 256; /* tokens, for their own form of the second product */
constexpr int kRank = 256, kSide = 1 << 24, kTokens = 16 * 65535;

const char *shape_error(const le_adapters *ad, int m) {
    if (ad->n_ad <= 0 || ad->rank <= 0 || ad->rank > kRank) return "n_ad below 1 or rank outside 1..256";
    if (ad->rows <= 0 || ad->cols <= 0 || ad->rows > kSide || ad->cols > kSide) return "rows or cols outside 1..2^24";
    if (m < 0 || m > kTokens) return "m outside 0..1048560";
    return nullptr;
}

/* How a call is cut up. */
struct Shape {
    int tiles, turns, sets, waves, segs, steps;
    size_t wave_lds;
    Shape(const le_adapters *ad, int xtype, int m) {
        tiles = (m + 15) / 16;
        /* blocks that share a tile's adapters: one each while there are few tiles (65 tokens with an adapter each 9 us, a block a tile 36); with
         * many, two, since most tiles have one or two (4096 tokens of 4096 values in runs of 456, rank 64: one 51, two 34, four 33 us) */
        turns = tiles <= 32 ? std::min(m, 16) : tiles <= 64 ? 4 : 2;
        /* of 16 rows of A at once (rank 64, two / four: 4096 tokens bf16 31 / 23 us, 64 tokens 7 / 6, fp32 17 / 13) */
        sets = ad->rank <= 16 ? 1 : ad->rank <= 32 ? 2 : 4;
        /* the columns' steps of 64 over a block's waves: eight, or as many as leave LDS for two blocks (few tokens: one, where fp32 rows
         * take most: 22 tokens of 20949 columns 21 / 31 us, 64 of 4096 11 / 13); four where every CU has a tile anyway (4 / 8
         * waves, 4096 tokens in runs of 456: fp32 34 / 40 us, bf16 23 / 26, 16384 of 1024 columns 14 / 18; 2048 tokens: 61 / 45). And over segments
         * while that makes no more than 2048 waves: up to eight for few tokens, each with an adapter of its own; for many, whose sums each of the second
         * kernel's row blocks reads again, two up to 1024 waves (1 / 2 / 4 segments, both kernels: 300 tokens 30 / 27 / 29 us, 1024 35 / 32 / 39,
         * 2048 45 / 53 / 54). */
        const int all = (ad->cols + 63) / 64;
        wave_lds = le_type_bytes(xtype) * 1024 + 256 + sets * (le_type_bytes(ad->ltype) * 1024 + 256);
        waves = std::min(std::min(tiles < 256 ? 8 : 4, (int)((m <= kFew ? 160 : 80) * 1024 / wave_lds)), all);
        segs = m <= kFew ? std::min(8, 2048 / (tiles * turns * waves)) : std::min(2, 1024 / (tiles * waves));
        segs = std::max(1, std::min(segs, all / waves));
        steps = (all + segs - 1) / segs;
        segs = (all + steps - 1) / steps;
    }
    size_t workspace(const le_adapters *ad) const { return (size_t)segs * tiles * ((ad->rank + 31) / 32) * 2048; }
};

}  // namespace

extern "C" size_t le_lora_workspace_size(const le_adapters *ad, int xtype, int m) {
    if (!ad || !le_type_bytes(xtype) || !le_type_bytes(ad->ltype) || shape_error(ad, m)) return 0;
    return m ? Shape(ad, xtype, m).workspace(ad) : 0;
}

extern "C" int le_lora(le_ctx *c, const le_adapters *ad, const int *idx, int xtype, const void *x, long long ldx, int m,
                       const void *base, long long ldb, void *y, long long ldy, void *ws, size_t ws_bytes, le_stream_t stream) {
    if (!c) return LE_ERR_ARG;
    if (!ad) return le_ctx_fail(c, LE_ERR_ARG, "null pointer");
    const int xb = le_type_bytes(xtype), wb = le_type_bytes(ad->ltype);
    if (!xb) return le_ctx_failf(c, LE_ERR_TYPE, "activations of type %d", xtype);
    if (!wb) return le_ctx_failf(c, LE_ERR_TYPE, "adapters of type %d", ad->ltype);
    if (const char *e = shape_error(ad, m))
        return le_ctx_failf(c, LE_ERR_SHAPE, "%s (%d adapters of rank %d, %d x %d, %d tokens)", e, ad->n_ad, ad->rank, ad->rows, ad->cols, m);
    if ((ldx && ldx < ad->cols) || (base && ldb < ad->rows) || ldy < ad->rows)
        return le_ctx_failf(c, LE_ERR_SHAPE, "row strides %lld, %lld and %lld of %d and %d values", ldx, ldb, ldy, ad->cols, ad->rows);
    if (m == 0) return LE_OK;
    if (!ad->a || !ad->b || !idx || !x || !y) return le_ctx_fail(c, LE_ERR_ARG, "null pointer");
    if (!le_aligned(ad->a, wb) || !le_aligned(ad->b, wb) || !le_aligned(ad->scale, 4) || !le_aligned(idx, 4) || !le_aligned(x, xb) ||
        !le_aligned(base, xb) || !le_aligned(y, xb) || !le_aligned(ws, 16))
        return le_ctx_fail(c, LE_ERR_ALIGN, "pointers must be aligned to their types, ws to 16 bytes");
    if (base == y && ldb != ldy) return le_ctx_fail(c, LE_ERR_ARG, "y in place of base has its row stride");
    const size_t need = le_lora_workspace_size(ad, xtype, m);
    if (!ws || ws_bytes < need) return le_ctx_failf(c, LE_ERR_WORKSPACE, "workspace needs %zu bytes", need);
    if (int rc = le_ctx_on_device(c)) return rc;
    const Shape sh(ad, xtype, m);
    LoraArgs a{ad->a, ad->b, ad->scale, idx, x, base, y, (float *)ws, ldx, ldb, ldy, ad->n_ad, ad->rank, ad->rows, ad->cols, m, sh.segs, sh.steps};
    void *args[] = {&a};
    char name[40];
    snprintf(name, sizeof name, "le_lo_down%d_%d_%d", sh.sets, xtype, ad->ltype);
    if (int rc = le_ctx_launch(c, name, dim3((unsigned)sh.tiles, (unsigned)sh.turns, (unsigned)sh.segs), 64 * sh.waves,
                               sh.waves * std::max(sh.wave_lds, (size_t)sh.sets * 1024), (hipStream_t)stream, args))
        return rc;
    const unsigned blocks = (unsigned)((ad->rows + 255) / 256);
    /* many tokens: a matrix instruction's 16 tokens at once, which pays where they have one adapter (4096 x 4096, rank 64 bf16, few / many form: 256
     * tokens in runs of 100 22 / 11 us, of 8 19 / 20, of one 45 / 84; 512 tokens 40 / 12, 31 / 21, 67 / 88) */
    if (m <= kFew) {
        int G = 1; /* lanes a row of B */
        while (8 * G < ad->rank) G *= 2;
        snprintf(name, sizeof name, "le_lo_upv%d_%d_%d", G, xtype, ad->ltype);
        return le_ctx_launch(c, name, dim3(std::min(blocks, (unsigned)std::max(1, 2048 / (sh.tiles * sh.turns))), (unsigned)sh.tiles, (unsigned)sh.turns), 256, 0, (hipStream_t)stream, args);
    }
    snprintf(name, sizeof name, "le_lo_upm%d_%d_%d", ad->rank % 8 || ad->rank > 64 ? 0 : ad->rank <= 32 ? 1 : 2, xtype, ad->ltype);
    return le_ctx_launch(c, name, dim3(blocks, (unsigned)((sh.tiles + 3) / 4)), 256, 0, (hipStream_t)stream, args);
}
