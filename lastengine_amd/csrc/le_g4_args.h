/* Kernel argument block of le_g4*, shared by host (le_g4.cpp) and device (le_g4_kernels.hip). */
#pragma once

struct G4Args {
    const unsigned char *codes;
    const void *scales, *zeros; /* zeros null: 8 */
    const int *sel;             /* null: slot s takes matrix s */
    const void *x;
    void *y;
    long long xstride; /* values */
    int n_mat, rows, cols, group, ng /* groups a row */, share, m;
    int gshift;        /* column >> gshift = group */
    int xty;           /* type of x and y */
    int nw, gx;        /* waves of a block, blocks of a slot (from here: the launch's own cost a load each) */
    unsigned char *ws; /* le_g4x_*, le_g4t_*, le_g4m_*: fragments of a set of m tokens */
    long long ws_set, ws_downs; /* bytes of a set, before its powers of two */
    float *part;               /* [segment of K][value of y], where there are several segments */
    long long total;           /* values of y */
    int segs, na;              /* na: le_g4t_*: sets of four virtual rows; 0: le_g4m_* */
    int per, full;     /* row groups of the blocks below `full`; the others have one less */
};
