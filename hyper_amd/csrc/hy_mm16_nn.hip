// Gradients of the rows: dz W, plain, of two parts and grouped by expert.
#include "hy_mm16_tile.cuh"

namespace hy {

template <typename T> static int tiles(const MMArgs &a, hipStream_t s, const char *what) {
    constexpr TileCost t[] = {T256x256, T128x128, T64x128, T64x64, T32x128, T32x64};
    switch (cheapest(t, a, NN, false)) {
    case 0: return launch_tile<T, NN, false, 256, 256, 2, 2, 2>(a, s, what);
    case 1: return launch_tile<T, NN, false, 128, 128, 2, 2, 2>(a, s, what);
    case 2: return launch_tile<T, NN, false, 64, 128, 2, 2, 3>(a, s, what);
    case 3: return launch_tile<T, NN, false, 64, 64, 2, 2, 4>(a, s, what);
    case 4: return launch_tile<T, NN, false, 32, 128, 4, 1, 3>(a, s, what);
    }
    return launch_tile<T, NN, false, 32, 64, 4, 1, 6>(a, s, what);
}
int launch_tiles_nn(int type, const MMArgs &a, hipStream_t s, const char *what) { return type == HY_BF16 ? tiles<bf16>(a, s, what) : tiles<f16>(a, s, what); }

} // namespace hy
