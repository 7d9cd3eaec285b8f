// Layer norm and RMS norm of rows, forward and backward.
//
// Forward: s = x (+ add), mu = mean(s) (RMS: 0), r = 1 / sqrt(mean((s - mu)^2) + eps), y = (s - mu) r w + b.  A row stays in the
// registers of the threads that loaded it, so the mean comes before the squares are summed; every value is read and written once.
// The mean is summed in 64 bits and taken from the rows as two floats, so that rows far from 0 beside their spread lose no more than
// a value's own rounding and equal values leave 0 (n <= 2^22 equal floats have a sum of at most 46 digits, and its quotient by n is
// exact).  As one float it would be off by up to half a step of the mean: rows of 1001 values around 1e5 with a spread of 0.05 had
// outputs off by up to 0.085 (so 6e-7).  That is what hy_norm_bwd gets, whose mean is one float.  All other sums are fp32.
// Backward: with h = (x - mu) r and g = dy w:  dx = r (g - mean(g) - h mean(g h)) + resid (RMS: without mean(g)),
// dw = sum over the rows of dy h, db = sum of dy.  A thread keeps its columns over all rows that its block takes, so dw and db
// are summed in registers, then over the block in LDS, and a second launch joins the blocks' sums in their order.
// Both are bound by their bytes where rows are many (8192 x 4096 fp32, RMS: with an added residual 81 us, 5.8 TB/s; backward 84 us,
// and 5 to join), by the launch where they are few (one row 2.4 us).
#include "hy_norm.cuh"

#include <algorithm>

namespace hy {

// A thread's 8 V values of a row that T threads share, in pieces of 16 bytes of the row's type X (PW = 4 or 8 neighbours): piece p at
// column PW (p T + t), so that neighbouring threads move neighbouring pieces (fp32 rows by 8 neighbours a thread instead: the
// gradient of 8192 x 4096 94 us for 86).
template <int T, int PW> __device__ __forceinline__ int norm_col(int t, int j, int i) { return PW * ((8 / PW * j + i / PW) * T + t) + i % PW; }
// PW neighbours wherever they start (the memory takes any alignment; rows of odd lengths one value at a time instead: 8192 x 4095
// bf16 142 us for 59)
template <typename Y, int PW> struct NeighboursOf { typedef Y vec __attribute__((ext_vector_type(PW))); typedef vec type __attribute__((aligned(sizeof(Y)))); };
template <typename Y, int PW> using Neighbours = typename NeighboursOf<Y, PW>::type;

// A row's last piece, and what would lie behind it, starts at n - PW instead, so that every load is a whole piece without a condition
// (values of their own each, by conditions, wait for each other: layer norm of bf16 16384 x 2047 93 us for 63, its gradient 98 for 56); the columns that
// come twice then are their first thread's, which norm_own says, and the other's copies are cleared before they enter a sum.  Rows
// shorter than a piece go by single values (PW = 1).
template <int T, int PW> __device__ __forceinline__ int norm_from(int t, int j, int h, int n) { return min(norm_col<T, PW>(t, j, h), n - PW); }
template <int T, int PW> __device__ __forceinline__ bool norm_own(int t, int j, int i, int n) {
    const int h = i - i % PW;
    return i % PW >= norm_col<T, PW>(t, j, h) - norm_from<T, PW>(t, j, h, n);
}
// a thread's values 8 j .. + 7 of a row of n values, n >= PW.  Y: the type of this row, whose columns go by PW
template <typename Y, int T, int PW> __device__ __forceinline__ void norm_load(const Y *row, int t, int j, int n, float (&v)[8]) {
#pragma unroll
    for (int h = 0; h < 8; h += PW) {
        const Neighbours<Y, PW> a = *(const Neighbours<Y, PW> *) (row + norm_from<T, PW>(t, j, h, n));
#pragma unroll
        for (int i = 0; i < PW; ++i) v[h + i] = (float) a[i];
    }
}
template <int T, int PW> __device__ __forceinline__ void norm_clear(int t, int j, int n, float (&v)[8]) {
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = norm_own<T, PW>(t, j, i, n) ? v[i] : 0.0f;
}
template <typename Y, int T, int PW> __device__ __forceinline__ void norm_store(Y *row, int t, int j, int n, const float (&v)[8]) {
#pragma unroll
    for (int h = 0; h < 8; h += PW) {
        const int c = norm_from<T, PW>(t, j, h, n);
        if (norm_own<T, PW>(t, j, h, n)) {
            Neighbours<Y, PW> a;
#pragma unroll
            for (int i = 0; i < PW; ++i) a[i] = (Y) v[h + i];
            *(Neighbours<Y, PW> *) (row + c) = a;
        } else {   // (its own alone: a row in place may not have been read by its other thread)
#pragma unroll
            for (int i = 1; i < PW; ++i) if (norm_own<T, PW>(t, j, h + i, n)) row[c + i] = (Y) v[h + i];
        }
    }
}
// the same where the type is known at run time only (the same for every thread)
template <int T, int PW> __device__ __forceinline__ void norm_load_as(int type, const void *base, int64_t at, int t, int j, int n, float (&v)[8]) {
    if (type == HY_F32) norm_load<float, T, PW>((const float *) base + at, t, j, n, v);
    else if (type == HY_BF16) norm_load<bf16, T, PW>((const bf16 *) base + at, t, j, n, v);
    else norm_load<f16, T, PW>((const f16 *) base + at, t, j, n, v);
}
template <int T, int PW> __device__ __forceinline__ void norm_store_as(int type, void *base, int64_t at, int t, int j, int n, const float (&v)[8]) {
    if (type == HY_F32) norm_store<float, T, PW>((float *) base + at, t, j, n, v);
    else if (type == HY_BF16) norm_store<bf16, T, PW>((bf16 *) base + at, t, j, n, v);
    else norm_store<f16, T, PW>((f16 *) base + at, t, j, n, v);
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

// the same in 64 bits, as two floats of the sum divided by n.  The steps of wave_sum_xor; vector double arithmetic runs at the rate of
// single here, and one sum in 64 bits takes the place of two in 32 (the mean, and the mean of what it left)
struct Mean2 { float hi, lo; };
template <int CTRL> __device__ __forceinline__ double dpp_d(double v) {
    const uint64_t b = (uint64_t) __double_as_longlong(v);
    const uint32_t lo = (uint32_t) dpp_i<CTRL>((int) (uint32_t) b), hi = (uint32_t) dpp_i<CTRL>((int) (uint32_t) (b >> 32));
    return __longlong_as_double((long long) ((uint64_t) hi << 32 | lo));
}
__device__ __forceinline__ double norm_lane_d(double v, int l) {
    const uint64_t b = (uint64_t) __double_as_longlong(v);
    const uint32_t lo = (uint32_t) __builtin_amdgcn_readlane((int) (uint32_t) b, l), hi = (uint32_t) __builtin_amdgcn_readlane((int) (uint32_t) (b >> 32), l);
    return __longlong_as_double((long long) ((uint64_t) hi << 32 | lo));
}
template <int T> __device__ __forceinline__ Mean2 row_mean(double v, int n, double *s) {
    v += dpp_d<DPP_XOR1>(v);
    v += dpp_d<DPP_XOR2>(v);
    v += dpp_d<DPP_HALF_MIRROR>(v);
    v += dpp_d<DPP_MIRROR>(v);
    v = (norm_lane_d(v, 0) + norm_lane_d(v, 16)) + (norm_lane_d(v, 32) + norm_lane_d(v, 48));
    if constexpr (T > 64) {
        if ((threadIdx.x & 63) == 0) s[(threadIdx.x % T) >> 6] = v;
        lds_barrier();
        v = 0.0;
#pragma unroll
        for (int i = 0; i < T / 64; ++i) v += s[i];
    }
    const double mu = v / (double) n;
    const float hi = (float) mu;
    return Mean2{hi, (float) (mu - (double) hi)};
}

constexpr int NORM_BLOCKS = 1 << 20;   // most blocks of a launch: they go on to further rows

// T threads a row of up to 8 V T values; a block has one row, or four of a wave each (T = 64: no barrier)
template <typename X, int T, int V, int PW = 16 / sizeof(X)> __global__ __launch_bounds__(T == 64 ? 256 : T) void k_norm(const NormArgs a) {
    constexpr int NT = T == 64 ? 256 : T, G = NT / T;
    __shared__ float s_sum[NT / 64];
    __shared__ double s_mean[NT / 64];
    const int t = threadIdx.x % T;
    for (int64_t row = (int64_t) blockIdx.x * G + threadIdx.x / T; row < a.m; row += (int64_t) gridDim.x * G) {
        float v[V][8];
#pragma unroll
        for (int j = 0; j < V; ++j) norm_load<X, T, PW>((const X *) a.x + row * a.ldx, t, j, a.n, v[j]);
        if (a.add) {
            float d[V][8];
#pragma unroll
            for (int j = 0; j < V; ++j) norm_load<X, T, PW>((const X *) a.add + row * a.lda, t, j, a.n, d[j]);
#pragma unroll
            for (int j = 0; j < V; ++j)
#pragma unroll
                for (int i = 0; i < 8; ++i) v[j][i] = (float) (X) (v[j][i] + d[j][i]);   // the sum as it stands in the stream
        }
#pragma unroll
        for (int j = 0; j < V; ++j) norm_clear<T, PW>(t, j, a.n, v[j]);
        if (a.total) {
#pragma unroll
            for (int j = 0; j < V; ++j) norm_store<X, T, PW>((X *) a.total + row * a.ldt, t, j, a.n, v[j]);
        }
        float q = 0.0f;
        Mean2 mu = {};
        if (a.layer) {
            double sum = 0.0;
#pragma unroll
            for (int j = 0; j < V; ++j)
#pragma unroll
                for (int i = 0; i < 8; ++i) sum += (double) v[j][i];
            mu = row_mean<T>(sum, a.n, s_mean);
#pragma unroll
            for (int j = 0; j < V; ++j)
#pragma unroll
                for (int i = 0; i < 8; ++i) v[j][i] = norm_own<T, PW>(t, j, i, a.n) ? (v[j][i] - mu.hi) - mu.lo : 0.0f;
        }
#pragma unroll
        for (int j = 0; j < V; ++j)
#pragma unroll
            for (int i = 0; i < 8; ++i) q = fmaf(v[j][i], v[j][i], q);
        const float r = 1.0f / sqrtf(row_sum<T>(q, s_sum) / (float) a.n + a.eps);
        if (t == 0) {
            if (a.mean) a.mean[row] = mu.hi;
            if (a.rstd) a.rstd[row] = r;
        }
#pragma unroll
        for (int j = 0; j < V; ++j) {
            if (norm_col<T, PW>(t, j, 0) >= a.n) continue;
            float w[8], y[8];
            norm_load<float, T, PW>(a.w, t, j, a.n, w);
            if (a.b) {
                float b[8];
                norm_load<float, T, PW>(a.b, t, j, a.n, b);
#pragma unroll
                for (int i = 0; i < 8; ++i) y[i] = fmaf(v[j][i] * r, w[i], b[i]);
            } else {
#pragma unroll
                for (int i = 0; i < 8; ++i) y[i] = v[j][i] * r * w[i];
            }
            if (a.out) norm_store_as<T, PW>(a.o_type, a.out, row * a.ldo, t, j, a.n, y);
            if (a.out32) norm_store<float, T, PW>(a.out32 + row * a.ldo32, t, j, a.n, y);
        }
        if constexpr (T > 64) lds_barrier();   // the sums are read before the next row's are written
    }
}

// the same for rows longer than a block's registers: passes over the row, whose later ones find it in the caches
template <typename X> __global__ __launch_bounds__(1024) void k_norm_long(const NormArgs a) {
    __shared__ float s_sum[16];
    __shared__ double s_mean[16];
    for (int64_t row = blockIdx.x; row < a.m; row += gridDim.x) {
        const X *x = (const X *) a.x + row * a.ldx, *d = a.add ? (const X *) a.add + row * a.lda : nullptr;
        X *tot = a.total ? (X *) a.total + row * a.ldt : nullptr;
        auto value = [&](int c) { return d ? (float) (X) ((float) x[c] + (float) d[c]) : (float) x[c]; };
        float q = 0.0f;
        Mean2 mu = {};
        if (a.layer) {
            double sum = 0.0;
            for (int c = threadIdx.x; c < a.n; c += 1024) sum += (double) value(c);
            mu = row_mean<1024>(sum, a.n, s_mean);
        }
        for (int c = threadIdx.x; c < a.n; c += 1024) { const float v = (value(c) - mu.hi) - mu.lo; q = fmaf(v, v, q); }
        const float r = 1.0f / sqrtf(row_sum<1024>(q, s_sum) / (float) a.n + a.eps);
        if (threadIdx.x == 0) {
            if (a.mean) a.mean[row] = mu.hi;
            if (a.rstd) a.rstd[row] = r;
        }
        for (int c = threadIdx.x; c < a.n; c += 1024) {
            const float s = value(c), v = ((s - mu.hi) - mu.lo) * r, y = a.b ? fmaf(v, a.w[c], a.b[c]) : v * a.w[c];
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

template <typename X> static void launch_norm_t(const NormArgs &a, hipStream_t s) {
    auto grid = [&](int rows) { return dim3((uint32_t) std::min<int64_t>(((int64_t) a.m + rows - 1) / rows, NORM_BLOCKS)); };
#define HY_NORM(T, V) k_norm<X, T, V><<<grid(T == 64 ? 4 : 1), T == 64 ? 256 : T, 0, s>>>(a)
    if (a.n > 16384) { k_norm_long<X><<<grid(1), 1024, 0, s>>>(a); return; }
    // 8 values a thread: a row in the registers of one wave (n 4096: 64 a thread) keeps too few rows of a CU under way (RMS of fp32
    // 8192 x 4096: 64 values a thread 114 us, 32 95, 16 85, 8 82; layer norm 16 98, 8 84).  16-bit rows wait for their sums rather:
    // 16 values, half as many waves to join (layer norm 45 us for 48, 8192 x 4093 58 for 68).  Threads between the powers of two, so that
    // few have nothing (layer norm of bf16 6000 x 5000: 768 threads of 8 values 60 us, 1024 97; fp32 90 and 123; 30000 x 700: one wave
    // 33 us, two 38), and 512 where 1024 would leave one row a CU (4000 x 7168 bf16 42 us for 61, fp32 87 for 92; 2000 x 14001 bf16 59
    // for 67, fp32 92 for 95)
    constexpr bool HALF = sizeof(X) == 2;
    if (a.n < 16 / (int) sizeof(X)) { k_norm<X, 64, 1, 1><<<grid(4), 256, 0, s>>>(a); return; }
    if (a.n <= 512) HY_NORM(64, 1);
    else if (HALF && a.n <= 768) HY_NORM(64, 2);
    else if (a.n <= 1024) HY_NORM(128, 1);
    else if (HALF && a.n <= 1536) HY_NORM(192, 1);
    else if (a.n <= 2048) HY_NORM(256, 1);
    else if (a.n <= 2560) HY_NORM(320, 1);
    else if (a.n <= 4096) { if (HALF) HY_NORM(256, 2); else HY_NORM(512, 1); }
    else if (a.n <= 6144) HY_NORM(768, 1);
    else if (a.n <= 8192) HY_NORM(512, 2);
    else if (a.n <= 12288) HY_NORM(768, 2);
    else HY_NORM(512, 4);
#undef HY_NORM
}
int launch_norm(int x_type, const NormArgs &a, hipStream_t s) {
    if (x_type == HY_F32) launch_norm_t<float>(a, s);
    else if (x_type == HY_BF16) launch_norm_t<bf16>(a, s);
    else launch_norm_t<f16>(a, s);
    return check_launch("hy_norm");
}

// ------------------------------------------------------------------ backward

// 8 values a thread here too: 16 of them (and their sums, 16 or 32 more) leave one block a CU (8192 x 4096 fp32: 104 us for 87).
// Blocks: those that a CU holds at a time; more of them begin a second round and have more sums to join (layer norm, 8192 x 4096: fp32 512
// blocks 83 us, 768 86; bf16 512 57, 768 69; 16384 x 2047: fp32 512 84, bf16 512 57, 768 56; 4000 x 7168 bf16: 256 blocks of 1024
// threads 55 us, 512 66).  Rows between the powers of two have threads and blocks of their own size (20000 x 1200: 192 threads a row 53 us
// in fp32 and 38 in bf16, 256 58 and 38; 12000 x 2501: 320 threads 73 and 68, 512 78 and 74; 5000 x 6001: 768 threads 83 and 69, 1024
// 87 and 71).  From 8192 values on two or four pieces a thread (3000 x 9001: 83 and 67 us; as the longest rows are done 162 and 149).
constexpr int NB_LONG = 16384;    // longer rows take k_norm_dx_long and k_norm_dw_long
__host__ __device__ constexpr int nb_row_threads(int n) { return n <= 512 ? 64 : n <= 1024 ? 128 : n <= 2048 ? 256 : n <= 4096 ? 512 : 1024; }
constexpr int nb_many_row_threads(int n) { return n > 1024 && n <= 1536 ? 192 : n > 2048 && n <= 2560 ? 320 : (n > 4096 && n <= 6144) || (n > 8192 && n <= 12288) ? 768 : nb_row_threads(n); }
__host__ __device__ constexpr int nb_block_threads(int T) { return T == 192 ? 384 : T == 320 ? 320 : T < 512 ? 512 : T; }

int norm_bwd_parts(int m, int n, bool x32) {
    const int T = nb_many_row_threads(n), g = n > NB_LONG ? 16 : nb_block_threads(T) / T;
    return (int) std::min<int64_t>(((int64_t) m + g - 1) / g, n > 4096 ? 256 : x32 || T == 512 ? 512 : 768);
}

// T threads a row of up to 8 V T values, G rows at a time; block b of `blocks` takes rows G b .. + G - 1 of every G blocks.  SUMS: dw
// and db of the thread's columns over its rows
template <typename X, int T, int V, bool LAYER, bool SUMS, int PW> __device__ __forceinline__ void norm_bwd_rows(const NormBwdArgs &a, int blocks, float (&dw)[V][8], float (&db)[V][8]) {
    constexpr int NT = nb_block_threads(T), G = NT / T, W = T / 64;
    constexpr bool EARLY = sizeof(X) == 4 && V == 1;   // the residual with the row (else: the registers are another block's)
    __shared__ float s_sum[2][2][NT / 64];
    const int t = threadIdx.x % T, g = threadIdx.x / T, wave = threadIdx.x >> 6;
    int turn = 0;
    for (int64_t first = (int64_t) blockIdx.x * G; first < a.m; first += (int64_t) blocks * G, turn ^= 1) {
        const int64_t row = first + g;
        const bool on = row < a.m;   // (the other threads go along for the barriers)
        float x[V][8], dy[V][8], e[8] = {}, c1 = 0.0f, c2 = 0.0f, r = 0.0f, mu = 0.0f;
        if (on) {
            r = a.rstd[row];
            if (LAYER) mu = a.mean[row];
#pragma unroll
            for (int j = 0; j < V; ++j) norm_load<X, T, PW>((const X *) a.x + row * a.ldx, t, j, a.n, x[j]);
            asm volatile("" ::: "memory");   // (else these loads come behind dy's, whose types are waited for: bf16 8192 x 4096, RMS 53 us for 48)
#pragma unroll
            for (int j = 0; j < V; ++j) {
                norm_load_as<T, PW>(a.y_type, a.dy, row * a.ldy, t, j, a.n, dy[j]);
                norm_clear<T, PW>(t, j, a.n, dy[j]);
            }
            float w[8];
            if (V == 1) norm_load<float, T, PW>(a.w, t, 0, a.n, w);
            if (EARLY && a.resid) norm_load<X, T, PW>((const X *) a.resid + row * a.ldr, t, 0, a.n, e);
#pragma unroll
            for (int j = 0; j < V; ++j) {
                if (V > 1) norm_load<float, T, PW>(a.w, t, j, a.n, w);
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    const float h = (x[j][i] - mu) * r;
                    if (SUMS) dw[j][i] = fmaf(dy[j][i], h, dw[j][i]);
                    if (SUMS && LAYER) db[j][i] += dy[j][i];
                    x[j][i] = h;
                    dy[j][i] *= w[i];   // zeros where the column is another's
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
#pragma unroll
        for (int j = 0; j < V; ++j) {
            if (on && norm_col<T, PW>(t, j, 0) < a.n) {
                const float m1 = c1 / (float) a.n, m2 = c2 / (float) a.n;
                float o[8];
                if (!EARLY && a.resid) norm_load<X, T, PW>((const X *) a.resid + row * a.ldr, t, j, a.n, e);
#pragma unroll
                for (int i = 0; i < 8; ++i) o[i] = r * ((LAYER ? dy[j][i] - m1 : dy[j][i]) - x[j][i] * m2) + e[i];
                norm_store<X, T, PW>((X *) a.dx + row * a.ldd, t, j, a.n, o);
            }
        }
    }
}
template <typename X, int T, int V, bool LAYER, int PW = 16 / sizeof(X)> __global__ __launch_bounds__(nb_block_threads(T)) void k_norm_bwd(const NormBwdArgs a) {
    constexpr int NT = nb_block_threads(T), G = NT / T, COLS = 8 * V * T;
    __shared__ float s_join[G > 1 ? G * COLS : 1];
    const int t = threadIdx.x % T, g = threadIdx.x / T;
    float dw[V][8] = {}, db[V][8] = {};
    norm_bwd_rows<X, T, V, LAYER, true, PW>(a, gridDim.x, dw, db);
    // the block's sums: over its G rows, in their order
#pragma unroll
    for (int which = 0; which < (LAYER ? 2 : 1); ++which) {
        float *out = which ? a.db : a.dw;
        if (!out) continue;
        float *to = a.part ? a.part + ((int64_t) which * gridDim.x + blockIdx.x) * a.n : out;
        const bool acc = !a.part && a.accumulate;
        if constexpr (G > 1) {
            static_assert(V == 1, "");
            __syncthreads();
#pragma unroll
            for (int i = 0; i < 8; ++i) if (norm_own<T, PW>(t, 0, i, a.n)) s_join[g * COLS + norm_from<T, PW>(t, 0, i - i % PW, a.n) + i % PW] = which ? db[0][i] : dw[0][i];
            __syncthreads();
            for (int c = threadIdx.x; c < a.n; c += NT) {
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
                    const int c = norm_from<T, PW>(t, j, i - i % PW, a.n) + i % PW;
                    const float v = which ? db[j][i] : dw[j][i];
                    if (norm_own<T, PW>(t, j, i, a.n)) to[c] = acc ? to[c] + v : v;
                }
        }
    }
}

// Few rows: the sums over the rows by blocks of their own beside the rows' blocks, each 32 columns and every 16th row a thread, so that
// one launch does (a second costs 3.5 us of the calling thread).  They read x and dy once more.
__device__ __forceinline__ float norm_value(int type, const void *base, int64_t at) {
    return type == HY_F32 ? ((const float *) base)[at] : type == HY_BF16 ? (float) ((const bf16 *) base)[at] : (float) ((const f16 *) base)[at];
}
template <typename X, int T, bool LAYER, int PW = 16 / sizeof(X)> __global__ __launch_bounds__(512) void k_norm_bwd_few(const NormBwdArgs a, int blocks) {
    static_assert(nb_block_threads(T) == 512, "");
    if ((int) blockIdx.x < blocks) {
        float none[1][8];
        norm_bwd_rows<X, T, 1, LAYER, false, PW>(a, blocks, none, none);
        return;
    }
    __shared__ float s[2][16][32];
    const int c = threadIdx.x & 31, g = threadIdx.x >> 5, col = ((int) blockIdx.x - blocks) * 32 + c;
    float dw = 0.0f, db = 0.0f;
    auto sum = [&](auto *dys) {
        const X *x = (const X *) a.x + col;
        for (int r0 = g; r0 < a.m; r0 += 16 * 8) {   // eight rows' values on their way together
            float xv[8], dv[8], rv[8], mv[8];
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const int row = min(r0 + 16 * i, a.m - 1);
                xv[i] = (float) x[row * a.ldx];
                dv[i] = (float) dys[row * a.ldy + col];
                rv[i] = a.rstd[row];
                mv[i] = LAYER ? a.mean[row] : 0.0f;
            }
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const bool in = r0 + 16 * i < a.m;
                dw = in ? fmaf(dv[i], (xv[i] - mv[i]) * rv[i], dw) : dw;
                if (LAYER) db += in ? dv[i] : 0.0f;
            }
        }
    };
    if (col < a.n) {
        if (a.y_type == HY_F32) sum((const float *) a.dy);
        else if (a.y_type == HY_BF16) sum((const bf16 *) a.dy);
        else sum((const f16 *) a.dy);
    }
    s[0][g][c] = dw;
    s[1][g][c] = db;
    __syncthreads();
    float *out = g == 0 ? a.dw : g == 1 && LAYER ? a.db : nullptr;
    if (out && col < a.n) {
        float v = 0.0f;
#pragma unroll
        for (int i = 0; i < 16; ++i) v += s[g][i][c];
        out[col] = a.accumulate ? out[col] + v : v;
    }
}

// rows longer than a block's registers: dx by one block a row in two passes ...
template <typename X> __global__ __launch_bounds__(1024) void k_norm_dx_long(const NormBwdArgs a) {
    __shared__ float s_sum[2][16];
    for (int64_t row = blockIdx.x; row < a.m; row += gridDim.x) {
        const X *x = (const X *) a.x + row * a.ldx;
        const float r = a.rstd[row], mu = a.mean ? a.mean[row] : 0.0f;
        float c1 = 0.0f, c2 = 0.0f;
        for (int c = threadIdx.x; c < a.n; c += 1024) {
            const float g = norm_value(a.y_type, a.dy, row * a.ldy + c) * a.w[c];
            c1 += g;
            c2 = fmaf(g, ((float) x[c] - mu) * r, c2);
        }
        c1 = a.mean ? row_sum<1024>(c1, s_sum[0]) / (float) a.n : 0.0f;
        c2 = row_sum<1024>(c2, s_sum[1]) / (float) a.n;
        for (int c = threadIdx.x; c < a.n; c += 1024) {
            const float g = norm_value(a.y_type, a.dy, row * a.ldy + c) * a.w[c], h = ((float) x[c] - mu) * r;
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
        const float dy = norm_value(a.y_type, a.dy, row * a.ldy + c), mu = a.mean ? a.mean[row] : 0.0f;
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

// Calls that k_norm_bwd_few is faster for, microseconds a call among others, fp16 layer norm and fp32 RMS: 509 x 1001 14.7 (k_norm_bwd and
// k_norm_join 17.4) and 12.5 (15.1); 1000 x 2048 14.6 (16.7) and 12.6 (15.2); 1000 x 4096 17.5 (29.9) and 18.4 (15.9); 2000 x 1001
// 19.8 (16.7) and 18.0 (15.3)
static bool norm_bwd_few(const NormBwdArgs &a, int x_bytes) {
    return a.parts > 1 && (a.dw || a.db) && a.m <= 1024 && a.n <= 4096 && a.m * a.n * x_bytes <= 1 << 23;
}
template <typename X, bool LAYER> static void launch_norm_bwd_t(const NormBwdArgs &a, hipStream_t s) {
    const dim3 grid(a.parts);
    const int n = a.n, PW = 16 / (int) sizeof(X);
    if (norm_bwd_few(a, sizeof(X))) {
        const int T = nb_row_threads(n), g = nb_block_threads(T) / T, blocks = (a.m + g - 1) / g, cols = (n + 31) / 32;
        auto go = [&](int rows, int all) {   // `rows` blocks of rows, then those of columns
            if (n < PW) k_norm_bwd_few<X, 64, LAYER, 1><<<all, 512, 0, s>>>(a, rows);
            else if (T == 64) k_norm_bwd_few<X, 64, LAYER><<<all, 512, 0, s>>>(a, rows);
            else if (T == 128) k_norm_bwd_few<X, 128, LAYER><<<all, 512, 0, s>>>(a, rows);
            else if (T == 256) k_norm_bwd_few<X, 256, LAYER><<<all, 512, 0, s>>>(a, rows);
            else k_norm_bwd_few<X, 512, LAYER><<<all, 512, 0, s>>>(a, rows);
        };
        if (a.dx != a.x && a.dx != a.dy) go(blocks, blocks + cols);
        else { go(0, cols); go(blocks, blocks); }   // dx takes the place of what the columns' blocks read: after them
        return;
    }
#define HY_NB(T, V) k_norm_bwd<X, T, V, LAYER><<<grid, nb_block_threads(T), 0, s>>>(a)
    switch (nb_many_row_threads(n)) {
    case 64: if (n < PW) k_norm_bwd<X, 64, 1, LAYER, 1><<<grid, 512, 0, s>>>(a); else HY_NB(64, 1); break;
    case 128: HY_NB(128, 1); break;
    case 192: HY_NB(192, 1); break;
    case 256: HY_NB(256, 1); break;
    case 320: HY_NB(320, 1); break;
    case 512: HY_NB(512, 1); break;
    case 768: if (n <= 6144) HY_NB(768, 1); else HY_NB(768, 2); break;
    default:
        if (n <= 8192) HY_NB(1024, 1);
        else if constexpr (LAYER && sizeof(X) == 4) k_norm_bwd<X, 512, 4, LAYER><<<grid, 512, 0, s>>>(a);   // (1024 threads have too few registers)
        else HY_NB(1024, 2);
    }
#undef HY_NB
}
template <typename X> static void launch_norm_bwd_x(bool layer, const NormBwdArgs &a, hipStream_t s) {
    if (a.n > NB_LONG) {
        if (a.dw || a.db) k_norm_dw_long<X><<<dim3((a.n + 255) / 256, a.parts), 256, 0, s>>>(a);
        k_norm_dx_long<X><<<(uint32_t) std::min(a.m, NORM_BLOCKS), 1024, 0, s>>>(a);
    } else if (layer) launch_norm_bwd_t<X, true>(a, s);
    else launch_norm_bwd_t<X, false>(a, s);
}
int launch_norm_bwd(int x_type, bool layer, const NormBwdArgs &a, hipStream_t s) {
    const char *what = "hy_norm_bwd";
    if (a.m == 0) {
        if (!a.accumulate && (a.dw || a.db)) k_norm_zero<<<(uint32_t) std::min((a.n + 255) / 256, 4096), 256, 0, s>>>(a.dw, a.db, a.n);
        return check_launch(what);
    }
    if (x_type == HY_F32) launch_norm_bwd_x<float>(layer, a, s);
    else if (x_type == HY_BF16) launch_norm_bwd_x<bf16>(layer, a, s);
    else launch_norm_bwd_x<f16>(layer, a, s);
    if (const int rc = check_launch(what)) return rc;
    if (a.part && (a.dw || a.db) && !norm_bwd_few(a, x_type == HY_F32 ? 4 : 2)) {
        k_norm_join<<<dim3((a.n + 63) / 64, a.db ? 2 : 1), 1024, 0, s>>>(a.part, a.parts, a.n, a.dw, a.db, a.accumulate);
        return check_launch(what);
    }
    return HY_OK;
}

} // namespace hy
