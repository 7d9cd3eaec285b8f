// Norms of rows, forward and backward: what the launchers and the kernels share.
#pragma once
#include "hy_mm16.cuh"

namespace hy {

// Types are HY_F32, HY_F16 or HY_BF16: x_type of x, add, total (backward: x, resid, dx), o_type of out (backward: dy)
struct NormArgs {
    const void *x, *add;
    void *total, *out;
    float *out32;
    const float *w, *b;
    float *mean, *rstd;
    int64_t ldx, lda, ldt, ldo, ldo32;
    int m, n, o_type;
    float eps;
    bool layer;   // subtract the mean
};
struct NormBwdArgs {
    const void *x, *dy, *resid;
    void *dx;
    const float *w, *mean, *rstd;
    float *dw, *db;
    float *part;   // [parts][n] sums of dw, then of db; null where one block has all rows
    int64_t ldx, ldy, ldr, ldd;
    int m, n, y_type, parts;
    bool accumulate;
};
int launch_norm(int x_type, const NormArgs &a, hipStream_t s);
int norm_bwd_parts(int m, int n, bool x32);   // (the most with false)
int launch_norm_bwd(int x_type, bool layer, const NormBwdArgs &a, hipStream_t s);

} // namespace hy
