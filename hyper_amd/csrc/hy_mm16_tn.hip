// Gradients of the weights: dz^T x, plain and grouped by expert.
#include "hy_mm16_tile.cuh"

namespace hy {

template <typename T> static int tiles(const MMArgs &a, hipStream_t s, const char *what) {
    if (a.R > 128 && a.N > 128) return launch_tile<T, TN, false, 256, 256, 2, 2, 2>(a, s, what);
    return launch_tile<T, TN, false, 128, 128, 2, 2, 2>(a, s, what);
}
int launch_tiles_tn(int type, const MMArgs &a, hipStream_t s, const char *what) { return type == HY_BF16 ? tiles<bf16>(a, s, what) : tiles<f16>(a, s, what); }

} // namespace hy
