// 16-bit products of few rows (single tokens), and the elementwise kernels around the products.
#include "hy_mm16.cuh"

#include <algorithm>

namespace hy {

// eight values at element offset `at` of a row of K values, zeros behind its end; AL: 16-byte aligned and K a multiple of 8
template <typename T, bool AL> __device__ __forceinline__ v8<T> ld8(const T *row, int at, int K) {
    if constexpr (AL) {
        v8<T> v = {};
        if (at < K) v = *(const v8<T> *) (row + at);
        return v;
    } else {
        v8<T> v = {};
        for (int i = 0; i < 8; ++i) if (at + i < K) v[i] = row[at + i];
        return v;
    }
}

// One wave for CW neighbouring columns and NR rows: lane l takes values 8 l .. + 7 of every 512 of the contraction.  By ids:
// blockIdx.y is a pair with its expert; else one group of a.R <= NR rows.  Bound by the weights' bytes.
template <typename T, bool DUAL, int NR, bool AL> __global__ __launch_bounds__(256) void k_mv(const MMArgs a) {
    constexpr int CW = DUAL ? 1 : 2;
    const int lane = threadIdx.x & 63;
    const int64_t col = ((int64_t) blockIdx.z * gridDim.x + blockIdx.x) * (4 * CW) + (threadIdx.x >> 6) * CW;
    if (col >= a.N) return;
    const int c0 = (int) col;
    int le = 0, row0 = 0, out0 = 0, nr = a.R;
    if (a.ids) {
        const int p = blockIdx.y, e = a.ids[p];
        if ((uint32_t) e >= (uint32_t) a.n_expert) return;
        le = a.slot[e];
        if ((uint32_t) le >= (uint32_t) a.n_local) return;
        row0 = div_k(p, a.kq);
        out0 = p;
        nr = 1;
    }
    const T *P = (const T *) a.P + (int64_t) le * a.pstride, *P2 = (const T *) a.P2 + (int64_t) le * a.pstride;
    const T *w[2];
    w[0] = P + (int64_t) c0 * a.ldp;
    w[1] = DUAL ? P2 + (int64_t) c0 * a.ldp : P + (int64_t) min(c0 + 1, a.N - 1) * a.ldp;
    const T *q[NR];
#pragma unroll
    for (int r = 0; r < NR; ++r) q[r] = (const T *) a.Q + (int64_t) (row0 + min(r, nr - 1)) * a.ldq;
    float acc[2][NR] = {};
    for (int k = lane * 8; k < a.K; k += 512) {
        const v8<T> w0 = ld8<T, AL>(w[0], k, a.K), w1 = ld8<T, AL>(w[1], k, a.K);
#pragma unroll
        for (int r = 0; r < NR; ++r) {
            const v8<T> x = ld8<T, AL>(q[r], k, a.K);
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                acc[0][r] = fmaf((float) w0[i], (float) x[i], acc[0][r]);
                acc[1][r] = fmaf((float) w1[i], (float) x[i], acc[1][r]);
            }
        }
    }
#pragma unroll
    for (int j = 0; j < 2; ++j)
#pragma unroll
        for (int r = 0; r < NR; ++r)
#pragma unroll
            for (int o = 32; o > 0; o >>= 1) acc[j][r] += __shfl_xor(acc[j][r], o);
    // lane r finishes row r
#pragma unroll
    for (int r = 0; r < NR; ++r) {
        if (lane != r || r >= nr) continue;
        const int64_t row = out0 + r;
        if constexpr (DUAL) {
            const int64_t at = row * a.ldo + c0;
            if (a.g) { ((T *) a.g)[at] = (T) acc[0][r]; ((T *) a.u)[at] = (T) acc[1][r]; }
            mm_limit<1>(&acc[0][r], &acc[1][r], a.clamp);
            ((T *) a.out)[at] = (T) mm_swiglu(acc[0][r], acc[1][r]);
        } else {
            const float wt = a.wts ? a.wts[row] : 1.0f;
#pragma unroll
            for (int j = 0; j < 2; ++j) {
                const int c = c0 + j;
                if (c >= a.N) break;
                float v = acc[j][r];
                if (a.bias) v += a.bias[c];
                if (a.z) ((T *) a.z)[row * a.ldz + c] = (T) v;
                if (a.act) v = mm_act(a.act, v);
                if (a.wts) v *= wt;
                if (a.resid) v += a.out_f32 ? ((const float *) a.resid)[row * a.ldr + c] : (float) ((const T *) a.resid)[row * a.ldr + c];
                if (a.out_f32) ((float *) a.out)[row * a.ldo + c] = v;
                else ((T *) a.out)[row * a.ldo + c] = (T) v;
            }
        }
    }
}

constexpr uint32_t MAX_ROW = 1 << 22;   // blocks in a row of the grid (a launch counts its threads in each direction in 32 bits)

template <typename T, bool DUAL, bool AL> static void mv_rows(const MMArgs &a, dim3 grid, hipStream_t s) {
    const int nr = a.ids ? 1 : a.R;
    if (nr == 1) k_mv<T, DUAL, 1, AL><<<grid, 256, 0, s>>>(a);
    else if (nr == 2) k_mv<T, DUAL, 2, AL><<<grid, 256, 0, s>>>(a);
    else k_mv<T, DUAL, 4, AL><<<grid, 256, 0, s>>>(a);
}
template <typename T> static int launch_mv_t(bool dual, const MMArgs &a, hipStream_t s, const char *what) {
    const bool al = a.K % 8 == 0 && a.ldp % 8 == 0 && a.ldq % 8 == 0 && a.pstride % 8 == 0 &&
                    (((uintptr_t) a.P | (uintptr_t) a.P2 | (uintptr_t) a.Q) & 15) == 0;
    const uint32_t blocks = (uint32_t) (dual ? (a.N + 3) / 4 : (a.N + 7) / 8), rows = (blocks + MAX_ROW - 1) / MAX_ROW;
    const dim3 grid(std::min(blocks, MAX_ROW), a.ids ? (uint32_t) a.n_pairs : 1u, rows);
    if (dual) { if (al) mv_rows<T, true, true>(a, grid, s); else mv_rows<T, true, false>(a, grid, s); }
    else { if (al) mv_rows<T, false, true>(a, grid, s); else mv_rows<T, false, false>(a, grid, s); }
    return check_launch(what);
}
int launch_mv(int type, bool dual, const MMArgs &a, hipStream_t s, const char *what) {
    return type == HY_BF16 ? launch_mv_t<bf16>(dual, a, s, what) : launch_mv_t<f16>(dual, a, s, what);
}

// ------------------------------------------------------------------ a few rows

static __device__ __attribute__((aligned(16))) const uint32_t g_zeros[4] = {0, 0, 0, 0};

// x W^T of up to 16 rows: a block of eight waves for 16 columns, the waves taking 64 of every 512 values of the contraction, straight
// to the registers of 16 x 16 x 32 products, four steps ahead; their sums meet in LDS.  Bound by the weights' bytes and, with them,
// each block's reads of x from L2 (5 rows of 4096 x 4096: 9.5 us, 3.5 TB/s of weights; 16 rows: 11.2 us).
template <typename T> __global__ __launch_bounds__(512) void k_few(const MMArgs a) {
    constexpr int DEPTH = 4;
    __shared__ f4 s_sum[8][64];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane((int) threadIdx.x >> 6), c0 = (int) blockIdx.x * 16;
    const int kl = wave * 64 + (lane >> 4) * 8;   // the lane's first value of a step's first half
    // (columns and rows outside are never stored)
    const T *w = (const T *) a.P + min(c0 + (lane & 15), a.N - 1) * a.ldp + kl, *x = (const T *) a.Q + min(lane & 15, a.R - 1) * a.ldq + kl;
    f4 acc = {};
    v8<T> fw[DEPTH][2], fx[DEPTH][2];
    auto load = [&](int d, int k) {   // k: the step's first value (a multiple of 512)
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            const bool in = k + kl + h * 32 < a.K;   // (K is a multiple of 8, and at most 2^30)
            fw[d][h] = *(const v8<T> *) (in ? w + k + h * 32 : (const T *) g_zeros);
            fx[d][h] = *(const v8<T> *) (in ? x + k + h * 32 : (const T *) g_zeros);
        }
    };
#pragma unroll
    for (int d = 0; d < DEPTH; ++d) load(d, d * 512);
    for (int k = 0; k < a.K; k += 512 * DEPTH) {
#pragma unroll
        for (int d = 0; d < DEPTH; ++d) {
#pragma unroll
            for (int h = 0; h < 2; ++h) acc = mfma16(fw[d][h], fx[d][h], acc);
            load(d, k + (DEPTH + d) * 512);
        }
    }
    s_sum[wave][lane] = acc;
    __syncthreads();
    if (wave) return;
    float v[4] = {};
#pragma unroll
    for (int u = 0; u < 8; ++u)
#pragma unroll
        for (int e = 0; e < 4; ++e) v[e] += s_sum[u][lane][e];
    if ((lane & 15) < a.R) epi_store<T, 4>(a, 0, lane & 15, c0 + (lane >> 4) * 4, v, 1.0f);
}

// One block a CU.  Microseconds, k_mv or tiles against k_few: 2 rows of 4096 x 14336 29.2 / 30.4, of 7168 x 4096 14.7 / 16.9; 4 rows of
// 4096 x 4096 12.2 / 9.5; 16 rows of 1024 x 2048, 4096 x 4096, 4096 x 14336 8.4 / 6.3, 14.5 / 11.2, 50 / 37, of 7168 x 4096 (448 blocks)
// 19.9 / 21.6.  32 rows (two row fragments) 15.8 / 15.7; gated (two fragments of columns, half the blocks) 14.7 / 15.4.
bool few_rows(const MMArgs &a) {
    return a.R >= 3 && a.R <= 16 && a.N <= 16 * 256 && a.K % 8 == 0 && a.ldp % 8 == 0 && a.ldq % 8 == 0 && (((uintptr_t) a.P | (uintptr_t) a.Q) & 15) == 0;
}
int launch_few(int type, const MMArgs &a, hipStream_t s, const char *what) {
    const uint32_t grid = (uint32_t) ((a.N + 15) / 16);
    if (type == HY_BF16) k_few<bf16><<<grid, 512, 0, s>>>(a);
    else k_few<f16><<<grid, 512, 0, s>>>(a);
    return check_launch(what);
}

// ------------------------------------------------------------------ elementwise

// dz = dy act'(z): eight values a thread where rows allow it (V = 8), else one
template <typename T, int V> __global__ __launch_bounds__(256) void k_act_bwd(int act, const T *z, int64_t ldz, const T *dy, int64_t lddy,
                                                                            int m, int n, T *dz, int64_t lddz) {
    const int per = (n + V - 1) / V;
    const int64_t total = (int64_t) m * per;
    for (int64_t i = (int64_t) blockIdx.x * 256 + threadIdx.x; i < total; i += (int64_t) gridDim.x * 256) {
        const int64_t r = i / per;
        const int c = (int) (i - r * per) * V;
        T zv[V], dv[V], o[V];
        if constexpr (V == 8) {
            *(v8<T> *) zv = *(const v8<T> *) (z + r * ldz + c);
            *(v8<T> *) dv = *(const v8<T> *) (dy + r * lddy + c);
        } else { zv[0] = z[r * ldz + c]; dv[0] = dy[r * lddy + c]; }
#pragma unroll
        for (int j = 0; j < V; ++j) o[j] = (T) ((float) dv[j] * mm_act_grad(act, (float) zv[j]));
        if constexpr (V == 8) *(v8<T> *) (dz + r * lddz + c) = *(v8<T> *) o;
        else dz[r * lddz + c] = o[0];
    }
}
template <typename T> static int launch_act_bwd_t(int act, const void *z, int64_t ldz, const void *dy, int64_t lddy, int m, int n, void *dz,
                                                  int64_t lddz, hipStream_t s) {
    const bool v = n % 8 == 0 && ldz % 8 == 0 && lddy % 8 == 0 && lddz % 8 == 0 && (((uintptr_t) z | (uintptr_t) dy | (uintptr_t) dz) & 15) == 0;
    const int64_t total = (int64_t) m * (v ? n / 8 : n);
    const uint32_t grid = (uint32_t) std::min<int64_t>((total + 255) / 256, 256 * 32);
    if (v) k_act_bwd<T, 8><<<grid, 256, 0, s>>>(act, (const T *) z, ldz, (const T *) dy, lddy, m, n, (T *) dz, lddz);
    else k_act_bwd<T, 1><<<grid, 256, 0, s>>>(act, (const T *) z, ldz, (const T *) dy, lddy, m, n, (T *) dz, lddz);
    return check_launch("hy_act_bwd");
}
int launch_act_bwd(int type, int act, const void *z, int64_t ldz, const void *dy, int64_t lddy, int m, int n, void *dz, int64_t lddz,
                   hipStream_t s) {
    return type == HY_BF16 ? launch_act_bwd_t<bf16>(act, z, ldz, dy, lddy, m, n, dz, lddz, s)
                           : launch_act_bwd_t<f16>(act, z, ldz, dy, lddy, m, n, dz, lddz, s);
}

// Gradient of w silu(g') u', g' = min(g, L), u' = clamp(u, -L, L) (L 0: none), one wave a pair:
//   hw = w h,  dg = w dh u' s (1 + g' (1 - s)) where g <= L,  du = w dh silu(g') where |u| <= L,  dwts = sum dh h
template <typename T, int V> __global__ __launch_bounds__(256) void k_swiglu_bwd(const T *g, const T *u, const T *dh, const float *wts,
                                                                               int n_pairs, int ff, float L, const int *order,
                                                                               const int *order_n, T *dg, T *du, T *hw, float *dwts) {
    const int lane = threadIdx.x & 63, i = (int) (blockIdx.y * gridDim.x + blockIdx.x) * 4 + (int) (threadIdx.x >> 6);
    int p = i;
    if (order) {
        if (i >= min(order_n[0], n_pairs)) return;
        p = order[i];
    }
    if ((uint32_t) p >= (uint32_t) n_pairs) return;
    const float w = wts ? wts[p] : 1.0f;
    const int64_t row = (int64_t) p * ff;
    float sum = 0.0f;
    for (int c = lane * V; c < ff; c += 64 * V) {
        T gv[V], uv[V], dv[V], og[V], ou[V], oh[V];
        if constexpr (V == 8) {
            *(v8<T> *) gv = *(const v8<T> *) (g + row + c);
            *(v8<T> *) uv = *(const v8<T> *) (u + row + c);
            *(v8<T> *) dv = *(const v8<T> *) (dh + row + c);
        } else { gv[0] = g[row + c]; uv[0] = u[row + c]; dv[0] = dh[row + c]; }
#pragma unroll
        for (int j = 0; j < V; ++j) {
            float gg = (float) gv[j], uu = (float) uv[j];
            const float d = (float) dv[j];
            bool gin = true, uin = true;
            if (L > 0.0f) {
                gin = !(gg > L);
                uin = !(uu > L || uu < -L);
                gg = gin ? gg : L;   // (NaN stays)
                uu = uin ? uu : copysignf(L, uu);
            }
            const float s = mm_sigmoid(gg), silu = gg * s, h = silu * uu;
            sum = fmaf(d, h, sum);
            oh[j] = (T) (w * h);
            og[j] = (T) (gin ? w * d * uu * fmaf(silu, 1.0f - s, s) : 0.0f);
            ou[j] = (T) (uin ? w * d * silu : 0.0f);
        }
        if constexpr (V == 8) {
            *(v8<T> *) (dg + row + c) = *(v8<T> *) og;
            *(v8<T> *) (du + row + c) = *(v8<T> *) ou;
            if (hw) *(v8<T> *) (hw + row + c) = *(v8<T> *) oh;
        } else {
            dg[row + c] = og[0];
            du[row + c] = ou[0];
            if (hw) hw[row + c] = oh[0];
        }
    }
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) sum += __shfl_xor(sum, o);
    if (dwts && lane == 0) dwts[p] = sum;
}
template <typename T> static int launch_swiglu_bwd_t(const void *g, const void *u, const void *dh, const float *wts, int n_pairs, int ff,
                                                     float clamp, const int *order, const int *order_n, void *dg, void *du, void *hw,
                                                     float *dwts, hipStream_t s) {
    const bool v = ff % 8 == 0 && (((uintptr_t) g | (uintptr_t) u | (uintptr_t) dh | (uintptr_t) dg | (uintptr_t) du | (uintptr_t) hw) & 15) == 0;
    const uint32_t blocks = (uint32_t) ((n_pairs + 3) / 4);
    const dim3 grid(std::min(blocks, MAX_ROW), (blocks + MAX_ROW - 1) / MAX_ROW);
    if (v) k_swiglu_bwd<T, 8><<<grid, 256, 0, s>>>((const T *) g, (const T *) u, (const T *) dh, wts, n_pairs, ff, clamp, order, order_n, (T *) dg, (T *) du, (T *) hw, dwts);
    else k_swiglu_bwd<T, 1><<<grid, 256, 0, s>>>((const T *) g, (const T *) u, (const T *) dh, wts, n_pairs, ff, clamp, order, order_n, (T *) dg, (T *) du, (T *) hw, dwts);
    return check_launch("hy_swiglu_bwd");
}
int launch_swiglu_bwd(int type, const void *g, const void *u, const void *dh, const float *wts, int n_pairs, int ff, float clamp,
                      const int *order, const int *order_n, void *dg, void *du, void *hw, float *dwts, hipStream_t s) {
    return type == HY_BF16 ? launch_swiglu_bwd_t<bf16>(g, u, dh, wts, n_pairs, ff, clamp, order, order_n, dg, du, hw, dwts, s)
                           : launch_swiglu_bwd_t<f16>(g, u, dh, wts, n_pairs, ff, clamp, order, order_n, dg, du, hw, dwts, s);
}

// fp32 rows rounded to T
template <typename T, int V> __global__ __launch_bounds__(256) void k_rows16(const float *x, int64_t xs, int n, int nt, T *out, int64_t ldo) {
    const int per = (n + V - 1) / V;
    const int64_t total = (int64_t) nt * per;
    for (int64_t i = (int64_t) blockIdx.x * 256 + threadIdx.x; i < total; i += (int64_t) gridDim.x * 256) {
        const int64_t r = i / per;
        const int c = (int) (i - r * per) * V;
        if constexpr (V == 4) {
            const f4 v = *(const f4 *) (x + r * xs + c);
            *(v4<T> *) (out + r * ldo + c) = v4<T>{(T) v[0], (T) v[1], (T) v[2], (T) v[3]};
        }
        else out[r * ldo + c] = (T) x[r * xs + c];
    }
}
template <typename T> static int launch_rows16_t(const float *x, int64_t xs, int n, int nt, void *out, int64_t ldo, hipStream_t s) {
    const bool v = n % 4 == 0 && xs % 4 == 0 && ldo % 4 == 0 && ((uintptr_t) x & 15) == 0 && ((uintptr_t) out & 7) == 0;
    const uint32_t grid = (uint32_t) std::min<int64_t>(((int64_t) nt * (v ? n / 4 : n) + 255) / 256, 256 * 32);
    if (v) k_rows16<T, 4><<<grid, 256, 0, s>>>(x, xs, n, nt, (T *) out, ldo);
    else k_rows16<T, 1><<<grid, 256, 0, s>>>(x, xs, n, nt, (T *) out, ldo);
    return check_launch("hy_rows16");
}
int launch_rows16(int type, const float *x, int64_t xs, int n, int nt, void *out, int64_t ldo, hipStream_t s) {
    return type == HY_BF16 ? launch_rows16_t<bf16>(x, xs, n, nt, out, ldo, s) : launch_rows16_t<f16>(x, xs, n, nt, out, ldo, s);
}

} // namespace hy
