// Forward products: x W^T, plain, gated and grouped by expert.
#include "hy_mm16_tile.cuh"

namespace hy {

template <typename T, bool DUAL> static int tiles(const MMArgs &a, hipStream_t s, const char *what) {
    // rows a group: all of them, or the pairs' share
    const int64_t rows = a.egrp ? a.n_pairs / std::max(1, std::min(a.max_active, a.n_expert)) : a.R;
    if (rows > 128) return launch_tile<T, NT, DUAL, 256, 256, 2, 2, 2>(a, s, what);
    if (rows > 48) return launch_tile<T, NT, DUAL, 128, 128, 2, 2, 2>(a, s, what);
    return launch_tile<T, NT, DUAL, 32, 128, 4, 1, 3>(a, s, what);
}
int launch_tiles_nt(int type, bool dual, const MMArgs &a, hipStream_t s, const char *what) {
    if (type == HY_BF16) return dual ? tiles<bf16, true>(a, s, what) : tiles<bf16, false>(a, s, what);
    return dual ? tiles<f16, true>(a, s, what) : tiles<f16, false>(a, s, what);
}

} // namespace hy
