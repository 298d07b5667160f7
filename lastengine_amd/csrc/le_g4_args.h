/* Kernel argument block of le_g4_*, shared by host (le_g4.cpp) and device (le_g4_kernels.hip). */
#pragma once

struct G4Args {
    const unsigned char *codes;
    const void *scales, *zeros; /* zeros null: 8 */
    const int *sel;             /* null: slot s takes matrix s */
    const void *x;
    void *y;
    long long xstride; /* values */
    int n_mat, rows, cols, group, ng /* groups a row */, share, m;
};
