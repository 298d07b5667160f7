/* Kernel argument block of the low-rank adapters, shared by host (le_lora.cpp) and device (le_lora_kernels.hip). */
#pragma once

struct LoraArgs {
    const void *a, *b;
    const float *scale; /* null: 1 */
    const int *idx;
    const void *x, *base; /* base null: 0 */
    void *y;
    float *u;             /* [segment][token][rank]: A x over a segment of the columns */
    long long ldx, ldb, ldy;
    int n_ad, rank, rows, cols, m;
    int segs, steps; /* segments of cols, the 64-column steps of each */
};
