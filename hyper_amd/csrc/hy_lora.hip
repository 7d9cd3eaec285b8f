// Low-rank adapters of many requests beside a shared projection: out[t] = resid[t] + scale_a B_a (A_a x[t]), a = ids[t].
//
// Two launches: the low products A_a x (r values a row, fp32, the contraction cut into parts that the second launch adds up), and
// B_a times them with the epilogue.  Both take 16 rows a matrix instruction and go through the adapters that occur among them
// one at a time; a row keeps the result of its own, so rows of any order and any mix of adapters are taken, and what other
// requests' matrices hold (NaN too) does not reach it.  Prompts have one or two adapters a tile; single tokens have up to 16, and
// then every product's weights are read for one row, which is what such a batch costs in any case: their bytes.
// The low products meet B as two 16-bit values each, rounded and rest, so that nothing of them is lost (one value alone would
// add half a step of the type to every product); fp16 takes them scaled by a power of two of its row, so that no value leaves
// its range.
#include "hy_lora.cuh"

#include <algorithm>

namespace hy {

// eight values of a row at column c, zeros behind its end; AL: the rows are whole 16-byte pieces
template <typename T, bool AL> __device__ __forceinline__ v8<T> lora_ld8(const T *row, int c, int end) {
    v8<T> v = {};
    if constexpr (AL) {
        if (c < end) v = *(const v8<T> *) (row + c);
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) if (c + i < end) v[i] = row[c + i];
    }
    return v;
}
// the adapter of lane i's row for lanes below ROWS, -1 where there is none
template <int ROWS> __device__ __forceinline__ int lora_id(const LoraArgs &a, int r0) {
    const int lane = threadIdx.x & 63;
    int id = -1;
    if (lane < ROWS && r0 + lane < a.m) id = a.ids[r0 + lane];
    return (uint32_t) id < (uint32_t) a.n_local ? id : -1;
}

// Low products of 16 rows over part blockIdx.y of the contraction, RT tiles of 16 ranks at a time; the four waves take every
// fourth 64 values and are added up in LDS.  A lane's 16 neighbouring values of a row are two products' operands (which of the
// contraction's values meet in which product does not matter as long as both operands agree), so that four lanes read 128
// neighbouring bytes.  The adapters of the tile are dealt out over blockIdx.z.
template <typename T, int RT, bool ALX, bool ALA> __global__ __launch_bounds__(256) void k_lora_low(const LoraArgs a) {
    __shared__ float s_acc[4][16][16 * RT + 4];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, q = lane >> 4, i16 = lane & 15;
    const int r0 = blockIdx.x * 16, k0 = blockIdx.y * a.klen, k1 = min(a.k, k0 + a.klen);
    const int id = lora_id<16>(a, r0);
    uint64_t left = __ballot(id >= 0);
    const T *xr = (const T *) a.x + (int64_t) min(r0 + i16, a.m - 1) * a.ldx;
    for (int turn = 0; left; ++turn) {
        const int ad = __builtin_amdgcn_readlane(id, __builtin_ctzll(left));
        const uint64_t mine = __ballot(id == ad);
        left &= ~mine;
        if (turn % gridDim.z != blockIdx.z) continue;
        for (int rb = 0; rb < a.r; rb += 16 * RT) {
            const T *A[RT];
#pragma unroll
            for (int j = 0; j < RT; ++j) A[j] = (const T *) a.A + ((int64_t) ad * a.r + min(rb + 16 * j + i16, a.r - 1)) * a.k;
            f4 acc[RT] = {};
            for (int kk = k0 + 64 * wave; kk < k1; kk += 256) {
                const int c = kk + 16 * q;
                const v8<T> x0 = lora_ld8<T, ALX>(xr, c, k1), x1 = lora_ld8<T, ALX>(xr, c + 8, k1);
                v8<T> a0[RT], a1[RT];
#pragma unroll
                for (int j = 0; j < RT; ++j) { a0[j] = lora_ld8<T, ALA>(A[j], c, k1); a1[j] = lora_ld8<T, ALA>(A[j], c + 8, k1); }
#pragma unroll
                for (int j = 0; j < RT; ++j) { acc[j] = mfma16(a0[j], x0, acc[j]); acc[j] = mfma16(a1[j], x1, acc[j]); }
            }
#pragma unroll
            for (int j = 0; j < RT; ++j) *(f4 *) &s_acc[wave][i16][16 * j + 4 * q] = acc[j];
            __syncthreads();
            for (int i = threadIdx.x; i < 16 * 16 * RT; i += 256) {
                const int row = i / (16 * RT), c = i % (16 * RT);
                if ((mine >> row & 1) && rb + c < a.r)
                    a.low[((int64_t) blockIdx.y * a.m + r0 + row) * a.r + rb + c] = (s_acc[0][row][c] + s_acc[1][row][c]) + (s_acc[2][row][c] + s_acc[3][row][c]);
            }
            __syncthreads();
        }
    }
}

// out of 16 RT rows x 256 columns, 64 columns a wave.  A lane holds 16 neighbouring columns of a row: column tile j's operand row i
// is column 16 (i / 4) + 4 j + i % 4.  R: the rank rounded up to 32, as the LDS rows hold it.
template <typename T, int RT, int R, bool ALB> __global__ __launch_bounds__(256) void k_lora_up(const LoraArgs a) {
    constexpr int LD = R + 8, ROWS = 16 * RT;
    __shared__ __attribute__((aligned(16))) T s_hi[ROWS * LD], s_lo[ROWS * LD];
    __shared__ float s_scale[ROWS];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, q = lane >> 4, i16 = lane & 15;
    const int r0 = blockIdx.x * ROWS, c0 = (blockIdx.y * 4 + wave) * 64;
    const int id = lora_id<ROWS>(a, r0);
    // the adapters of the tile that are this block's: their rows
    uint64_t left = __ballot(id >= 0), rows = 0;
    for (int turn = 0; left; ++turn) {
        const uint64_t mine = __ballot(id == __builtin_amdgcn_readlane(id, __builtin_ctzll(left)));
        left &= ~mine;
        if (turn % gridDim.z == blockIdx.z) rows |= mine;
    }
    // their low products, four threads a row and 32 ranks
    constexpr int TPR = 256 / ROWS, PER = R / TPR;   // threads a row, values a thread
    {
        const int row = threadIdx.x / TPR, t = threadIdx.x % TPR;
        float v[PER], top = 0.0f;
#pragma unroll
        for (int i = 0; i < PER; ++i) v[i] = 0.0f;
        if (rows >> row & 1) {
            const float *low = a.low + (int64_t) (r0 + row) * a.r;
            for (int sp = 0; sp < a.splits; ++sp, low += (int64_t) a.m * a.r)
#pragma unroll
                for (int i = 0; i < PER; ++i) if (t + TPR * i < a.r) v[i] += low[t + TPR * i];
        }
        float up = 1.0f;
        if constexpr (sizeof(T) == 2 && __is_same(T, f16)) {
#pragma unroll
            for (int i = 0; i < PER; ++i) top = fmaxf(top, fabsf(v[i]));
#pragma unroll
            for (int o = 1; o < TPR; o <<= 1) top = fmaxf(top, __shfl_xor(top, o));
            const int e = (int) (__float_as_uint(top) >> 23) - 127;   // 2^e <= top
            if (top < __builtin_huge_valf() && e > -100) up = __uint_as_float((uint32_t) (127 + min(max(13 - e, -113), 113)) << 23);   // the largest to 2^13 .. 2^14
        }
        if (t == 0) s_scale[row] = 1.0f / up;
#pragma unroll
        for (int i = 0; i < PER; ++i) {
            const float u = v[i] * up;
            const T hi = (T) u;
            const float rest = u - (float) hi;
            s_hi[row * LD + t + TPR * i] = hi;
            s_lo[row * LD + t + TPR * i] = rest - rest == 0.0f ? (T) rest : (T) 0.0f;   // (none of an infinity)
        }
    }
    __syncthreads();
    if (c0 >= a.n) return;
    f4 out[RT][4] = {};
    left = rows;
    while (left) {
        const int ad = __builtin_amdgcn_readlane(id, __builtin_ctzll(left));
        const uint64_t mine = __ballot(id == ad);
        left &= ~mine;
        f4 acc[RT][4] = {};
#pragma unroll 1
        for (int kk = 0; kk < a.r; kk += 32) {
            v8<T> b[4];
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const int c = min(c0 + 16 * (i16 >> 2) + 4 * j + (i16 & 3), a.n - 1);
                b[j] = lora_ld8<T, ALB>((const T *) a.B + ((int64_t) ad * a.n + c) * a.r, kk + 8 * q, a.r);
            }
#pragma unroll
            for (int i = 0; i < RT; ++i) {
                if (!(mine >> (16 * i) & 0xffff)) continue;   // (the same in every lane)
                const v8<T> hi = *(const v8<T> *) &s_hi[(16 * i + i16) * LD + kk + 8 * q], lo = *(const v8<T> *) &s_lo[(16 * i + i16) * LD + kk + 8 * q];
#pragma unroll
                for (int j = 0; j < 4; ++j) { acc[i][j] = mfma16(b[j], lo, acc[i][j]); acc[i][j] = mfma16(b[j], hi, acc[i][j]); }
            }
        }
        const float sc = a.scale ? a.scale[ad] : 1.0f;
#pragma unroll
        for (int i = 0; i < RT; ++i) {
            if (!(mine >> (16 * i + i16) & 1)) continue;
            const float s = sc * s_scale[16 * i + i16];
#pragma unroll
            for (int j = 0; j < 4; ++j)
#pragma unroll
                for (int e = 0; e < 4; ++e) out[i][j][e] = acc[i][j][e] * s;
        }
    }
    // this block's rows; those without an adapter are the first blocks'
    const uint64_t none = __ballot(id < 0 && lane < ROWS && r0 + lane < a.m);
    const uint64_t write = blockIdx.z == 0 && !(a.resid == a.out && a.ldr == a.ldo) ? rows | none : rows;
#pragma unroll
    for (int i = 0; i < RT; ++i) {
        if (!(write >> (16 * i + i16) & 1)) continue;
        const int64_t row = r0 + 16 * i + i16;
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            const int c = c0 + 16 * q + 8 * h, n = min(8, a.n - c);
            if (n <= 0) continue;
            float v[8];
#pragma unroll
            for (int e = 0; e < 8; ++e) v[e] = out[i][2 * h + (e >> 2)][e & 3];
            if (a.resid) add_n<T, 8>(a.resid, row * a.ldr + c, v, n, a.out_f32, a.vec);
            put_n<T, 8>(a.out, row * a.ldo + c, v, n, a.out_f32, a.vec);
        }
    }
}

// Parts of at least 256 values of the contraction, as many as make 512 blocks of 16 rows
LoraCut lora_cut(int m, int k) {
    const int tiles = (m + 15) / 16, most = std::max(1, std::min(32, (k + 255) / 256));
    const int want = std::max(1, std::min(most, (512 + tiles - 1) / std::max(1, tiles)));
    const int klen = ((k + want - 1) / want + 255) / 256 * 256;
    return LoraCut{(int) (((int64_t) k + klen - 1) / klen), klen};
}

static bool lora_al(const void *p, int64_t ld) { return ((uintptr_t) p & 15) == 0 && ld % 8 == 0; }

template <typename T> static int launch_lora_t(const LoraArgs &a, hipStream_t s) {
    const char *what = "hy_lora";
    const int tiles = (a.m + 15) / 16;
    const bool alx = lora_al(a.x, a.ldx) && a.k % 8 == 0, ala = lora_al(a.A, a.k), alb = lora_al(a.B, a.r);
    const dim3 low(tiles, a.splits, std::max(1, std::min(16, 1024 / std::max(1, tiles * a.splits))));
#define HY_LOW(RT) { if (alx && ala) k_lora_low<T, RT, true, true><<<low, 256, 0, s>>>(a); \
                     else k_lora_low<T, RT, false, false><<<low, 256, 0, s>>>(a); }
    if (a.r <= 16) HY_LOW(1) else if (a.r <= 32) HY_LOW(2) else HY_LOW(4)
#undef HY_LOW
    if (const int rc = check_launch(what)) return rc;
    const int cols = (a.n + 255) / 256;
    const bool tall = a.r <= 64 && a.m >= 256;
    const int rt = tall ? (a.m + 63) / 64 : tiles;
    const dim3 up(rt, cols, std::max(1, std::min(16, 1024 / std::max(1, rt * cols))));
#define HY_UP(RT, R) { if (alb) k_lora_up<T, RT, R, true><<<up, 256, 0, s>>>(a); else k_lora_up<T, RT, R, false><<<up, 256, 0, s>>>(a); }
    if (a.r <= 32) { if (tall) HY_UP(4, 32) else HY_UP(1, 32) }
    else if (a.r <= 64) { if (tall) HY_UP(4, 64) else HY_UP(1, 64) }
    else if (a.r <= 128) HY_UP(1, 128)
    else HY_UP(1, 256)
#undef HY_UP
    return check_launch(what);
}
int launch_lora(int type, const LoraArgs &a, hipStream_t s) { return type == HY_BF16 ? launch_lora_t<bf16>(a, s) : launch_lora_t<f16>(a, s); }

} // namespace hy
