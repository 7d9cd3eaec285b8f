// Gradients of the weights: dz^T x, plain and grouped by expert.
#include "hy_mm16_tile.cuh"

namespace hy {

template <typename T> static int tiles(const MMArgs &a, hipStream_t s, const char *what) {
    constexpr TileCost t[] = {T256x256, T128x128, T64x128};
    switch (cheapest(t, a, TN, false)) {
    case 0: return launch_tile<T, TN, false, 256, 256, 2, 2, 2>(a, s, what);
    case 1: return launch_tile<T, TN, false, 128, 128, 2, 2, 2>(a, s, what);
    }
    return launch_tile<T, TN, false, 64, 128, 2, 2, 3>(a, s, what);
}
int launch_tiles_tn(int type, const MMArgs &a, hipStream_t s, const char *what) { return type == HY_BF16 ? tiles<bf16>(a, s, what) : tiles<f16>(a, s, what); }

} // namespace hy
