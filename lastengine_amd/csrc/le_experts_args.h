/* Kernel argument block of the experts' products, shared by host (le_experts.cpp) and device (le_experts_kernels.hip). */
#pragma once

struct ExpertArgs {
    const void *a, *b; /* rows along M and N of the product; one of the two may be the weights */
    void *y;
    const int *off;
    long long lda, ldb, ldy; /* values */
    int n_exp, n_row;
    int m, n, k;     /* outputs and depth; the one that counts an expert's rows is n_row here */
    int mt, nt;      /* tiles along M (weights' gradient) and N */
    int run;         /* tiles in a row that one XCD takes */
    int segs;        /* weights' gradient: parts of an expert's rows, each with sums of its own */
    int strip;       /* few rows: tiles of 32 outputs that a wave takes one after the other */
};
