// Forward products: x W^T, plain, gated and grouped by expert.
#include "hy_mm16_tile.cuh"

namespace hy {

template <typename T, bool DUAL> static int tiles(const MMArgs &a, hipStream_t s, const char *what) {
    constexpr TileCost t[] = {T256x256, T128x128, T64x128, T64x64, T32x128, T32x64};
    constexpr int WP = DUAL ? 2 : 4, WQ = DUAL ? 2 : 1;   // 32 x 64: a gated wave takes 16 gate and 16 up columns
    switch (cheapest(t, a, NT, DUAL)) {
    case 0: return launch_tile<T, NT, DUAL, 256, 256, 2, 2, 2>(a, s, what);
    case 1: return launch_tile<T, NT, DUAL, 128, 128, 2, 2, 2>(a, s, what);
    case 2: return launch_tile<T, NT, DUAL, 64, 128, 2, 2, 3>(a, s, what);
    case 3: return launch_tile<T, NT, DUAL, 64, 64, 2, 2, 4>(a, s, what);
    case 4: return launch_tile<T, NT, DUAL, 32, 128, 4, 1, 3>(a, s, what);
    }
    return launch_tile<T, NT, DUAL, 32, 64, WP, WQ, 6>(a, s, what);
}
int launch_tiles_nt(int type, bool dual, const MMArgs &a, hipStream_t s, const char *what) {
    if (type == HY_BF16) return dual ? tiles<bf16, true>(a, s, what) : tiles<bf16, false>(a, s, what);
    return dual ? tiles<f16, true>(a, s, what) : tiles<f16, false>(a, s, what);
}

} // namespace hy
