/* Kernel argument block of le_add_rms_quant, shared by host (le_norm.cpp) and device (le_norm_kernels.hip). */
#pragma once

struct NormArgs {
    const void *x, *res; /* res null: none */
    const float *w;
    void *h, *o;         /* may be null */
    signed char *xq;     /* null with xd */
    float *xd;
    int *xs;             /* may be null */
    long long ldx, ldr, ldh, ldo;
    int m, n;
    float eps;
};
