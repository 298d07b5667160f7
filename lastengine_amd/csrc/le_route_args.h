/* Kernel argument blocks of the expert-routing kernels, shared by host (le_route.cpp) and device (le_route_kernels.hip). */
#pragma once

struct RouteArgs {
    const void *logits;
    int *idx;
    float *w;
    int n_tok, n_exp, k;
};
struct RouteBwdArgs {
    const int *idx;
    const float *w, *dw;
    void *dlogits;
    int n_tok, n_exp, k;
};
struct SortArgs {
    const int *idx;
    int *off, *in_idx, *out_idx, *pos; /* all but off may be null */
    int np, k, n_exp;
    int blocks, waves, steps; /* a wave takes 64 * steps pairs */
    int *ws;                  /* [block][expert] counts, where there are several blocks */
};
struct RowsArgs {
    const void *src;  /* permute: x; combine: e; backward: dout */
    const void *e;    /* backward: e (null where dw is) */
    void *dst;        /* permute: e; combine: out; backward: de (may be null) */
    const int *pos;   /* null: pos[p] = p */
    const float *w;   /* null: 1 */
    float *dw;        /* backward; may be null */
    long long ldt, lde;
    int n_tok, k, cols, n_row;
};
