// Gradients of the rows: dz W, plain, of two parts and grouped by expert.
#include "hy_mm16_tile.cuh"

namespace hy {

template <typename T> static int tiles(const MMArgs &a, hipStream_t s, const char *what) {
    const int64_t rows = a.egrp ? a.n_pairs / std::max(1, std::min(a.max_active, a.n_expert)) : a.R;
    if (rows > 128) return launch_tile<T, NN, false, 256, 256, 2, 2, 2>(a, s, what);
    if (rows > 48) return launch_tile<T, NN, false, 128, 128, 2, 2, 2>(a, s, what);
    return launch_tile<T, NN, false, 32, 128, 4, 1, 3>(a, s, what);
}
int launch_tiles_nn(int type, const MMArgs &a, hipStream_t s, const char *what) { return type == HY_BF16 ? tiles<bf16>(a, s, what) : tiles<f16>(a, s, what); }

} // namespace hy
