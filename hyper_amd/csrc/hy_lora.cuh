// Low-rank adapters of many requests at once: what the launchers and the kernels share.
#pragma once
#include "hy_mm16.cuh"

namespace hy {

struct LoraArgs {
    const void *A, *B, *x;
    const float *scale;
    const int *ids;
    const void *resid;
    void *out;
    float *low;      // [splits][m][r]: the splits' sums of A x
    int64_t ldx, ldr, ldo;
    int m, n, k, r, n_local;
    int splits, klen;   // the contraction cut into `splits` parts of klen values
    int out_f32;
};
struct LoraCut { int splits, klen; };
LoraCut lora_cut(int m, int k);
int launch_lora(int type, const LoraArgs &a, hipStream_t s);

} // namespace hy
