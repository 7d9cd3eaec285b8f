// Layer norm and RMS norm of rows, forward and backward.
//
// Forward: s = x (+ add), mu = mean(s) (RMS: 0), r = 1 / sqrt(mean((s - mu)^2) + eps), y = (s - mu) r w + b.  A row stays in the
// registers of the threads that loaded it, so the mean comes before the squares are summed, is corrected by the mean of
// what it leaves, and nothing cancels; every value is read and written once.  All sums are fp32.
// Backward: with h = (x - mu) r and g = dy w:  dx = r (g - mean(g) - h mean(g h)) + resid (RMS: without mean(g)),
// dw = sum over the rows of dy h, db = sum of dy.  A thread keeps its columns over all rows that its block takes, so dw and db
// are summed in registers, then over the block in LDS, and a second launch joins the blocks' sums in their order.
#include "hy_norm.cuh"

#include <algorithm>

namespace hy {

// A thread's V pieces of 8 values of a row that T threads share.  VEC: piece j is columns 8 (j T + t) .. + 7, moved in 16-byte
// pieces; else its value i is column (8 j + i) T + t, so that neighbouring threads touch neighbouring values.
template <int T, bool VEC> __device__ __forceinline__ int norm_col(int t, int j, int i) { return VEC ? 8 * (j * T + t) + i : (8 * j + i) * T + t; }

template <typename X> __device__ __forceinline__ void norm_ld8(const X *p, float (&v)[8]) {
    if constexpr (sizeof(X) == 4) {
        const f4 a = *(const f4 *) p, b = *(const f4 *) (p + 4);
#pragma unroll
        for (int i = 0; i < 4; ++i) { v[i] = a[i]; v[4 + i] = b[i]; }
    } else {
        const v8<X> a = *(const v8<X> *) p;
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = (float) a[i];
    }
}
template <typename X> __device__ __forceinline__ void norm_st8(X *p, const float (&v)[8]) {
    if constexpr (sizeof(X) == 4) {
        *(f4 *) p = f4{v[0], v[1], v[2], v[3]};
        *(f4 *) (p + 4) = f4{v[4], v[5], v[6], v[7]};
    } else {
        v8<X> a;
#pragma unroll
        for (int i = 0; i < 8; ++i) a[i] = (X) v[i];
        *(v8<X> *) p = a;
    }
}
// piece j of a row of n values, zeros behind its end
template <typename X, int T, bool VEC> __device__ __forceinline__ void norm_load(const X *row, int t, int j, int n, float (&v)[8]) {
    if constexpr (VEC) {
        const int c = norm_col<T, true>(t, j, 0);
        if (c + 8 <= n) { norm_ld8<X>(row + c, v); return; }
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const int c = norm_col<T, VEC>(t, j, i);
        v[i] = c < n ? (float) row[c] : 0.0f;
    }
}
template <typename X, int T, bool VEC> __device__ __forceinline__ void norm_store(X *row, int t, int j, int n, const float (&v)[8]) {
    if constexpr (VEC) {
        const int c = norm_col<T, true>(t, j, 0);
        if (c + 8 <= n) { norm_st8<X>(row + c, v); return; }
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const int c = norm_col<T, VEC>(t, j, i);
        if (c < n) row[c] = (X) v[i];
    }
}
// the same where the type is known at run time only (the same for every thread)
template <int T, bool VEC> __device__ __forceinline__ void norm_load_as(int type, const void *base, int64_t at, int t, int j, int n, float (&v)[8]) {
    if (type == HY_F32) norm_load<float, T, VEC>((const float *) base + at, t, j, n, v);
    else if (type == HY_BF16) norm_load<bf16, T, VEC>((const bf16 *) base + at, t, j, n, v);
    else norm_load<f16, T, VEC>((const f16 *) base + at, t, j, n, v);
}
template <int T, bool VEC> __device__ __forceinline__ void norm_store_as(int type, void *base, int64_t at, int t, int j, int n, const float (&v)[8]) {
    if (type == HY_F32) norm_store<float, T, VEC>((float *) base + at, t, j, n, v);
    else if (type == HY_BF16) norm_store<bf16, T, VEC>((bf16 *) base + at, t, j, n, v);
    else norm_store<f16, T, VEC>((f16 *) base + at, t, j, n, v);
}

// the sum of v over the T threads of a row; `s`: this row's T / 64 floats of LDS, written anew by each call
template <int T> __device__ __forceinline__ float row_sum(float v, float *s) {
    v = wave_sum_xor(v);
    if constexpr (T > 64) {
        if ((threadIdx.x & 63) == 0) s[(threadIdx.x % T) >> 6] = v;
        lds_barrier();
        v = 0.0f;
#pragma unroll
        for (int i = 0; i < T / 64; ++i) v += s[i];
    }
    return v;
}

constexpr int NORM_BLOCKS = 1 << 20;   // most blocks of a launch: they go on to further rows

// T threads a row of up to 8 V T values, max(T, 256) threads a block
template <typename X, int T, int V, bool VEC> __global__ __launch_bounds__(T < 256 ? 256 : T) void k_norm(const NormArgs a) {
    constexpr int NT = T < 256 ? 256 : T, G = NT / T;
    __shared__ float s_sum[3][NT / 64];
    const int t = threadIdx.x % T;
    for (int64_t row = (int64_t) blockIdx.x * G + threadIdx.x / T; row < a.m; row += (int64_t) gridDim.x * G) {
        float v[V][8];
#pragma unroll
        for (int j = 0; j < V; ++j) norm_load<X, T, VEC>((const X *) a.x + row * a.ldx, t, j, a.n, v[j]);
        if (a.add) {
            float d[V][8];
#pragma unroll
            for (int j = 0; j < V; ++j) norm_load<X, T, VEC>((const X *) a.add + row * a.lda, t, j, a.n, d[j]);
#pragma unroll
            for (int j = 0; j < V; ++j)
#pragma unroll
                for (int i = 0; i < 8; ++i) v[j][i] = (float) (X) (v[j][i] + d[j][i]);   // the sum as it stands in the stream
        }
        if (a.total) {
#pragma unroll
            for (int j = 0; j < V; ++j) norm_store<X, T, VEC>((X *) a.total + row * a.ldt, t, j, a.n, v[j]);
        }
        float mu = 0.0f, q = 0.0f;
        if (a.layer) {
#pragma unroll
            for (int j = 0; j < V; ++j)
#pragma unroll
                for (int i = 0; i < 8; ++i) mu += v[j][i];
            mu = row_sum<T>(mu, s_sum[0]) / (float) a.n;
            float e = 0.0f;   // what the sum's rounding left: rows far from 0 beside their spread keep it (equal values have none)
#pragma unroll
            for (int j = 0; j < V; ++j)
#pragma unroll
                for (int i = 0; i < 8; ++i) if (norm_col<T, VEC>(t, j, i) < a.n) e += v[j][i] - mu;
            mu += row_sum<T>(e, s_sum[2]) / (float) a.n;
        }
#pragma unroll
        for (int j = 0; j < V; ++j)
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                v[j][i] -= mu;
                if (norm_col<T, VEC>(t, j, i) < a.n) q = fmaf(v[j][i], v[j][i], q);
            }
        const float r = 1.0f / sqrtf(row_sum<T>(q, s_sum[1]) / (float) a.n + a.eps);
        if (t == 0) {
            if (a.mean) a.mean[row] = mu;
            if (a.rstd) a.rstd[row] = r;
        }
#pragma unroll
        for (int j = 0; j < V; ++j) {
            if (norm_col<T, VEC>(t, j, 0) >= a.n) continue;
            float w[8], y[8];
            norm_load<float, T, VEC>(a.w, t, j, a.n, w);
            if (a.b) {
                float b[8];
                norm_load<float, T, VEC>(a.b, t, j, a.n, b);
#pragma unroll
                for (int i = 0; i < 8; ++i) y[i] = fmaf(v[j][i] * r, w[i], b[i]);
            } else {
#pragma unroll
                for (int i = 0; i < 8; ++i) y[i] = v[j][i] * r * w[i];
            }
            if (a.out) norm_store_as<T, VEC>(a.o_type, a.out, row * a.ldo, t, j, a.n, y);
            if (a.out32) norm_store<float, T, VEC>(a.out32 + row * a.ldo32, t, j, a.n, y);
        }
        if constexpr (T > 64) lds_barrier();   // the sums are read before the next row's are written
    }
}

// the same for rows longer than a block's registers: passes over the row, whose later ones find it in the caches
template <typename X> __global__ __launch_bounds__(1024) void k_norm_long(const NormArgs a) {
    __shared__ float s_sum[3][16];
    for (int64_t row = blockIdx.x; row < a.m; row += gridDim.x) {
        const X *x = (const X *) a.x + row * a.ldx, *d = a.add ? (const X *) a.add + row * a.lda : nullptr;
        X *tot = a.total ? (X *) a.total + row * a.ldt : nullptr;
        auto value = [&](int c) { return d ? (float) (X) ((float) x[c] + (float) d[c]) : (float) x[c]; };
        float mu = 0.0f, q = 0.0f;
        if (a.layer) {
            for (int c = threadIdx.x; c < a.n; c += 1024) mu += value(c);
            mu = row_sum<1024>(mu, s_sum[0]) / (float) a.n;
            float e = 0.0f;
            for (int c = threadIdx.x; c < a.n; c += 1024) e += value(c) - mu;
            mu += row_sum<1024>(e, s_sum[2]) / (float) a.n;
        }
        for (int c = threadIdx.x; c < a.n; c += 1024) { const float v = value(c) - mu; q = fmaf(v, v, q); }
        const float r = 1.0f / sqrtf(row_sum<1024>(q, s_sum[1]) / (float) a.n + a.eps);
        if (threadIdx.x == 0) {
            if (a.mean) a.mean[row] = mu;
            if (a.rstd) a.rstd[row] = r;
        }
        for (int c = threadIdx.x; c < a.n; c += 1024) {
            const float s = value(c), v = (s - mu) * r, y = a.b ? fmaf(v, a.w[c], a.b[c]) : v * a.w[c];
            if (tot) tot[c] = (X) s;
            if (a.out) {
                if (a.o_type == HY_F32) ((float *) a.out)[row * a.ldo + c] = y;
                else if (a.o_type == HY_BF16) ((bf16 *) a.out)[row * a.ldo + c] = (bf16) y;
                else ((f16 *) a.out)[row * a.ldo + c] = (f16) y;
            }
            if (a.out32) a.out32[row * a.ldo32 + c] = y;
        }
        lds_barrier();
    }
}

template <typename X, bool VEC> static void launch_norm_t(const NormArgs &a, hipStream_t s) {
    auto grid = [&](int rows) { return dim3((uint32_t) std::min<int64_t>(((int64_t) a.m + rows - 1) / rows, NORM_BLOCKS)); };
#define HY_NORM(T, V) k_norm<X, T, V, VEC><<<grid(T < 256 ? 256 / T : 1), T < 256 ? 256 : T, 0, s>>>(a)
    if (a.n > 16384) { k_norm_long<X><<<grid(1), 1024, 0, s>>>(a); return; }
    if (a.n <= 512) HY_NORM(64, 1);
    else if (a.m >= 1024 && a.n <= 1024) HY_NORM(64, 2);
    else if (a.m >= 1024 && a.n <= 2048) HY_NORM(64, 4);
    else if (a.m >= 1024 && a.n <= 4096) HY_NORM(64, 8);
    else if (a.n <= 2048) HY_NORM(256, 1);
    else if (a.n <= 4096) HY_NORM(256, 2);
    else if (a.n <= 8192) { if (a.m >= 1024) HY_NORM(256, 4); else HY_NORM(1024, 1); }
    else HY_NORM(1024, 2);
#undef HY_NORM
}
int launch_norm(int x_type, const NormArgs &a, bool vec, hipStream_t s) {
    if (x_type == HY_F32) vec ? launch_norm_t<float, true>(a, s) : launch_norm_t<float, false>(a, s);
    else if (x_type == HY_BF16) vec ? launch_norm_t<bf16, true>(a, s) : launch_norm_t<bf16, false>(a, s);
    else vec ? launch_norm_t<f16, true>(a, s) : launch_norm_t<f16, false>(a, s);
    return check_launch("hy_norm");
}

// ------------------------------------------------------------------ backward

constexpr int NB_T = 512;         // threads a block: NB_T / T rows at a time
constexpr int NB_BLOCKS = 512;    // most blocks: two a CU
constexpr int NB_LONG = 8192;    // longer rows than this take k_norm_bwd_long

__host__ __device__ constexpr int nb_threads(int n) { return n <= 1024 ? 64 : n <= 4096 ? 256 : NB_T; }   // threads a row

int norm_bwd_parts(int m, int n) {
    const int g = n > NB_LONG ? 16 : NB_T / nb_threads(n);
    return (int) std::min<int64_t>(((int64_t) m + g - 1) / g, NB_BLOCKS);
}

// T threads a row, NB_T / T rows at a time; block b takes rows G b .. + G - 1 of every G gridDim.x
template <typename X, int T, int V, bool LAYER, bool VEC> __global__ __launch_bounds__(NB_T) void k_norm_bwd(const NormBwdArgs a) {
    constexpr int G = NB_T / T, W = T / 64, COLS = 8 * V * T;
    __shared__ float s_sum[2][2][NB_T / 64];
    __shared__ float s_join[G > 1 ? G * COLS : 1];
    const int t = threadIdx.x % T, g = threadIdx.x / T, wave = threadIdx.x >> 6;
    float dw[V][8] = {}, db[LAYER ? V : 1][8] = {};
    int turn = 0;
    for (int64_t first = (int64_t) blockIdx.x * G; first < a.m; first += (int64_t) gridDim.x * G, turn ^= 1) {
        const int64_t row = first + g;
        const bool on = row < a.m;   // (the other threads go along for the barriers)
        float x[V][8], dy[V][8], c1 = 0.0f, c2 = 0.0f, r = 0.0f, mu = 0.0f;
        if (on) {
            r = a.rstd[row];
            if (LAYER) mu = a.mean[row];
#pragma unroll
            for (int j = 0; j < V; ++j) norm_load<X, T, VEC>((const X *) a.x + row * a.ldx, t, j, a.n, x[j]);
#pragma unroll
            for (int j = 0; j < V; ++j) norm_load_as<T, VEC>(a.y_type, a.dy, row * a.ldy, t, j, a.n, dy[j]);
#pragma unroll
            for (int j = 0; j < V; ++j) {
                float w[8];
                norm_load<float, T, VEC>(a.w, t, j, a.n, w);
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    const float h = (x[j][i] - mu) * r;
                    dw[j][i] = fmaf(dy[j][i], h, dw[j][i]);
                    if (LAYER) db[j][i] += dy[j][i];
                    x[j][i] = h;
                    dy[j][i] *= w[i];   // zeros behind the row's end
                    if (LAYER) c1 += dy[j][i];
                    c2 = fmaf(dy[j][i], h, c2);
                }
            }
        }
        c2 = wave_sum_xor(c2);
        if (LAYER) c1 = wave_sum_xor(c1);
        if constexpr (W > 1) {
            if ((threadIdx.x & 63) == 0) { s_sum[turn][0][wave] = c2; if (LAYER) s_sum[turn][1][wave] = c1; }
            lds_barrier();   // (the next row's sums go to the other half: one barrier a row)
            c1 = c2 = 0.0f;
#pragma unroll
            for (int i = 0; i < W; ++i) { c2 += s_sum[turn][0][g * W + i]; if (LAYER) c1 += s_sum[turn][1][g * W + i]; }
        }
        if (on) {
            c1 /= (float) a.n;
            c2 /= (float) a.n;
#pragma unroll
            for (int j = 0; j < V; ++j) {
                if (norm_col<T, VEC>(t, j, 0) >= a.n) continue;
                float o[8];
#pragma unroll
                for (int i = 0; i < 8; ++i) o[i] = r * ((LAYER ? dy[j][i] - c1 : dy[j][i]) - x[j][i] * c2);
                if (a.resid) {
                    float e[8];
                    norm_load<X, T, VEC>((const X *) a.resid + row * a.ldr, t, j, a.n, e);
#pragma unroll
                    for (int i = 0; i < 8; ++i) o[i] += e[i];
                }
                norm_store<X, T, VEC>((X *) a.dx + row * a.ldd, t, j, a.n, o);
            }
        }
    }
    // the block's sums: over its G rows, in their order
#pragma unroll
    for (int which = 0; which < (LAYER ? 2 : 1); ++which) {
        float *out = which ? a.db : a.dw;
        if (!out) continue;
        float *to = a.part ? a.part + ((int64_t) which * gridDim.x + blockIdx.x) * a.n : out;
        const bool acc = !a.part && a.accumulate;
        if constexpr (G > 1) {
            __syncthreads();
#pragma unroll
            for (int j = 0; j < V; ++j)
#pragma unroll
                for (int i = 0; i < 8; ++i) s_join[g * COLS + norm_col<T, VEC>(t, j, i)] = which ? db[LAYER ? j : 0][i] : dw[j][i];
            __syncthreads();
            for (int c = threadIdx.x; c < a.n; c += NB_T) {
                float v = 0.0f;
#pragma unroll
                for (int k = 0; k < G; ++k) v += s_join[k * COLS + c];
                to[c] = acc ? to[c] + v : v;
            }
        } else {
#pragma unroll
            for (int j = 0; j < V; ++j)
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    const int c = norm_col<T, VEC>(t, j, i);
                    const float v = which ? db[LAYER ? j : 0][i] : dw[j][i];
                    if (c < a.n) to[c] = acc ? to[c] + v : v;
                }
        }
    }
}

// rows longer than a block's registers: dx by one block a row in two passes ...
template <typename X> __device__ __forceinline__ float dy_at(int type, const void *dy, int64_t at) {
    return type == HY_F32 ? ((const float *) dy)[at] : type == HY_BF16 ? (float) ((const bf16 *) dy)[at] : (float) ((const f16 *) dy)[at];
}
template <typename X> __global__ __launch_bounds__(1024) void k_norm_dx_long(const NormBwdArgs a) {
    __shared__ float s_sum[2][16];
    for (int64_t row = blockIdx.x; row < a.m; row += gridDim.x) {
        const X *x = (const X *) a.x + row * a.ldx;
        const float r = a.rstd[row], mu = a.mean ? a.mean[row] : 0.0f;
        float c1 = 0.0f, c2 = 0.0f;
        for (int c = threadIdx.x; c < a.n; c += 1024) {
            const float g = dy_at<X>(a.y_type, a.dy, row * a.ldy + c) * a.w[c];
            c1 += g;
            c2 = fmaf(g, ((float) x[c] - mu) * r, c2);
        }
        c1 = a.mean ? row_sum<1024>(c1, s_sum[0]) / (float) a.n : 0.0f;
        c2 = row_sum<1024>(c2, s_sum[1]) / (float) a.n;
        for (int c = threadIdx.x; c < a.n; c += 1024) {
            const float g = dy_at<X>(a.y_type, a.dy, row * a.ldy + c) * a.w[c], h = ((float) x[c] - mu) * r;
            const float v = r * (g - c1 - h * c2);
            ((X *) a.dx)[row * a.ldd + c] = (X) (a.resid ? v + (float) ((const X *) a.resid)[row * a.ldr + c] : v);
        }
        lds_barrier();
    }
}
// ... after the sums over the rows, a thread a column and blockIdx.y a part of the rows (dx may be x or dy)
template <typename X> __global__ __launch_bounds__(256) void k_norm_dw_long(const NormBwdArgs a) {
    const int64_t c = (int64_t) blockIdx.x * 256 + threadIdx.x;
    if (c >= a.n) return;
    float dw = 0.0f, db = 0.0f;
    for (int64_t row = blockIdx.y; row < a.m; row += gridDim.y) {
        const float dy = dy_at<X>(a.y_type, a.dy, row * a.ldy + c), mu = a.mean ? a.mean[row] : 0.0f;
        dw = fmaf(dy, ((float) ((const X *) a.x)[row * a.ldx + c] - mu) * a.rstd[row], dw);
        db += dy;
    }
    if (a.dw) { float *o = a.part ? a.part + (int64_t) blockIdx.y * a.n + c : a.dw + c; *o = !a.part && a.accumulate ? *o + dw : dw; }
    if (a.db) { float *o = a.part ? a.part + ((int64_t) gridDim.y + blockIdx.y) * a.n + c : a.db + c; *o = !a.part && a.accumulate ? *o + db : db; }
}

// the parts' sums of 64 columns, in a fixed order: 16 waves take every 16th part, then their sums in turn
__global__ __launch_bounds__(1024) void k_norm_join(const float *part, int parts, int n, float *dw, float *db, bool accumulate) {
    __shared__ float s[16][64];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    float *out = blockIdx.y ? db : dw;
    if (!out) return;
    const int64_t c = (int64_t) blockIdx.x * 64 + lane;
    const float *p = part + (int64_t) blockIdx.y * parts * n + c;
    float v = 0.0f;
    if (c < n) {
#pragma unroll 16
        for (int i = wave; i < parts; i += 16) v += p[(int64_t) i * n];
    }
    s[wave][lane] = v;
    __syncthreads();
    if (wave == 0 && c < n) {
        v = 0.0f;
#pragma unroll
        for (int i = 0; i < 16; ++i) v += s[i][lane];
        out[c] = accumulate ? out[c] + v : v;
    }
}
__global__ __launch_bounds__(256) void k_norm_zero(float *dw, float *db, int n) {
    for (int64_t c = (int64_t) blockIdx.x * 256 + threadIdx.x; c < n; c += (int64_t) gridDim.x * 256) {
        if (dw) dw[c] = 0.0f;
        if (db) db[c] = 0.0f;
    }
}

template <typename X, bool LAYER, bool VEC> static void launch_norm_bwd_t(const NormBwdArgs &a, hipStream_t s) {
    const dim3 grid(a.parts);
    const int n = a.n;
#define HY_NB(T, V) k_norm_bwd<X, T, V, LAYER, VEC><<<grid, NB_T, 0, s>>>(a)
    if (n <= 512) HY_NB(64, 1);
    else if (n <= 1024) HY_NB(64, 2);
    else if (n <= 2048) HY_NB(256, 1);
    else if (n <= 4096) HY_NB(256, 2);
    else HY_NB(512, 2);
#undef HY_NB
}
template <typename X> static void launch_norm_bwd_x(bool layer, const NormBwdArgs &a, bool vec, hipStream_t s) {
    if (a.n > NB_LONG) {
        if (a.dw || a.db) k_norm_dw_long<X><<<dim3((a.n + 255) / 256, a.parts), 256, 0, s>>>(a);
        k_norm_dx_long<X><<<(uint32_t) std::min(a.m, NORM_BLOCKS), 1024, 0, s>>>(a);
    } else if (layer) vec ? launch_norm_bwd_t<X, true, true>(a, s) : launch_norm_bwd_t<X, true, false>(a, s);
    else vec ? launch_norm_bwd_t<X, false, true>(a, s) : launch_norm_bwd_t<X, false, false>(a, s);
}
int launch_norm_bwd(int x_type, bool layer, const NormBwdArgs &a, bool vec, hipStream_t s) {
    const char *what = "hy_norm_bwd";
    if (a.m == 0) {
        if (!a.accumulate && (a.dw || a.db)) k_norm_zero<<<(uint32_t) std::min((a.n + 255) / 256, 4096), 256, 0, s>>>(a.dw, a.db, a.n);
        return check_launch(what);
    }
    if (x_type == HY_F32) launch_norm_bwd_x<float>(layer, a, vec, s);
    else if (x_type == HY_BF16) launch_norm_bwd_x<bf16>(layer, a, vec, s);
    else launch_norm_bwd_x<f16>(layer, a, vec, s);
    if (const int rc = check_launch(what)) return rc;
    if (a.part && (a.dw || a.db)) {
        k_norm_join<<<dim3((a.n + 63) / 64, a.db ? 2 : 1), 1024, 0, s>>>(a.part, a.parts, a.n, a.dw, a.db, a.accumulate);
        return check_launch(what);
    }
    return HY_OK;
}

} // namespace hy
