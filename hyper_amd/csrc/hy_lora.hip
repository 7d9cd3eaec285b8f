// Low-rank adapters of many requests beside a shared projection: out[t] = resid[t] + scale_a B_a (A_a x[t]), a = ids[t].
//
// Two launches: the low products A_a x (r values a row, fp32, the contraction cut into parts that the second launch adds up), and
// B_a times them with the epilogue.  Both take 16 rows a matrix instruction and go through the adapters that occur among them
// one at a time; a row keeps the result of its own, so rows of any order and any mix of adapters are taken, and what other
// requests' matrices hold (NaN too) does not reach it.  Prompts have one or two adapters a tile; single tokens have up to 16, and
// then every product's weights are read for one row, which is what such a batch costs in any case: their bytes.
// The low products, fp32, meet B as sums of 16-bit values, each the rounding of what those before it left; fp16 takes them scaled
// by a power of two of its row, so that no value leaves its range.  For 16-bit outputs two values: they keep a bf16 product within 2^-16
// of itself and an fp16 one within 2^-22 (or 2^-38 of its row's largest), beside 2^-8 and 2^-11 that the output is rounded by; one
// alone would add half a step of the type to every product.  For fp32 outputs three, which hold all 24 bits (with two: 4096 rows of 24
// prompts, 4096 -> 7168, rank 64, both launches 81 us for 82, rank 256 233 for 236; 1000 rows with an adapter each, rank 16, 45 for 46).
// Bound: single tokens by the launches and the latency of ids, operands and low products in turn (16 rows with an adapter each,
// rank 16, 4096 x 4096: 4.2 and 6.0 us); prompts by B and the residual on their way through the caches (4096 rows of 24 prompts,
// rank 64, 4096 -> 7168: 18.5 and 43 us, 155 MB in the second).
#include "hy_lora.cuh"

#include <algorithm>

namespace hy {

// N neighbours wherever they start: the memory takes any alignment (rows of odd lengths in single values instead: 4096 rows,
// 4096 -> 7161, rank 64, 303 us)
template <typename Y, int N> struct LoraVec { typedef Y vec __attribute__((ext_vector_type(N))); typedef vec type __attribute__((aligned(sizeof(Y)))); };
template <typename Y, int N> __device__ __forceinline__ typename LoraVec<Y, N>::vec lora_get(const Y *p) { return *(const typename LoraVec<Y, N>::type *) p; }
// N values of a row at column c, zeros behind its end
template <typename Y, int N> __device__ __forceinline__ typename LoraVec<Y, N>::vec lora_ld(const Y *row, int c, int end) {
    typename LoraVec<Y, N>::vec v = {};
    if (c + N <= end) v = lora_get<Y, N>(row + c);
    else {
#pragma unroll
        for (int i = 0; i < N; ++i) if (c + i < end) v[i] = row[c + i];
    }
    return v;
}
// Lanes 2 i and 2 i + 1 (neighbouring rows of an operand or output) exchange one 16-byte piece: the even lane keeps p and gives q,
// the odd lane keeps q and gives p.  Memory is then met eight lanes to a row and 128 bytes, as whole lines; a row's own four
// lanes alone meet 64 bytes (low products of 4096 rows of 4096 values, rank 64: 26 us for 20).
template <typename V> __device__ __forceinline__ void pair_swap(V &p, V &q) {
    static_assert(sizeof(V) == 16, "");
    typedef int i32x4 __attribute__((ext_vector_type(4)));
    const bool odd = threadIdx.x & 1;
    i32x4 a = __builtin_bit_cast(i32x4, p), b = __builtin_bit_cast(i32x4, q);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const int got = dpp_i<DPP_XOR1>(odd ? a[i] : b[i]);
        if (odd) a[i] = got; else b[i] = got;
    }
    p = __builtin_bit_cast(V, a);
    q = __builtin_bit_cast(V, b);
}
// the adapter of lane i's row for lanes below ROWS, -1 where there is none
template <int ROWS> __device__ __forceinline__ int lora_id(const LoraArgs &a, int r0) {
    const int lane = threadIdx.x & 63;
    int id = -1;
    if (lane < ROWS && r0 + lane < a.m) id = a.ids[r0 + lane];
    return (uint32_t) id < (uint32_t) a.n_local ? id : -1;
}

// Low products of 16 RW rows over a part of the contraction, RT tiles of 16 ranks at a time; the four waves take every
// fourth 64 values and are added up in LDS.  The adapters of the tile are dealt out over blockIdx.z.
template <typename T, int RT, int RW> struct LowStep {   // a step's operands; as loaded: piece 0 of the even row, piece 1 of the odd one
    v8<T> x[RW][2], w[RT][2];
    __device__ __forceinline__ void load(const T *const (&xr)[RW][2], const T *const (&A)[RT][2], int at) {
#pragma unroll
        for (int i = 0; i < RW; ++i) { x[i][0] = lora_get<T, 8>(xr[i][0] + at); x[i][1] = lora_get<T, 8>(xr[i][1] + at); }
#pragma unroll
        for (int j = 0; j < RT; ++j) { w[j][0] = lora_get<T, 8>(A[j][0] + at); w[j][1] = lora_get<T, 8>(A[j][1] + at); }
    }
    __device__ __forceinline__ void swap() {
#pragma unroll
        for (int i = 0; i < RW; ++i) pair_swap(x[i][0], x[i][1]);
#pragma unroll
        for (int j = 0; j < RT; ++j) pair_swap(w[j][0], w[j][1]);
    }
    __device__ __forceinline__ void add(f4 (&acc)[RW][RT]) const {
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
            for (int i = 0; i < RW; ++i)
#pragma unroll
                for (int j = 0; j < RT; ++j) acc[i][j] = mfma16(w[j][h], x[i][h], acc[i][j]);
    }
};
// Between the loads of a step and the products of the one before: else the compiler moves the loads to where they are used, and
// nothing is in flight while the products run
__device__ __forceinline__ void lora_keep_order() {
    asm volatile("" ::: "memory");
    __builtin_amdgcn_sched_barrier(0);
}
template <typename T, int RT, int RW> __global__ __launch_bounds__(256) void k_lora_low(const LoraArgs a) {
    __shared__ float s_acc[4][16][16 * RT + 4];
    constexpr int ROWS = 16 * RW, STEP = 256;   // (a wave's own 64 values, then the other waves')
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, q = lane >> 4, i16 = lane & 15;
    const int w = xcd_tile(blockIdx.x, gridDim.x), part = w % a.splits;   // neighbouring tiles on one XCD: they share adapters
    const int r0 = w / a.splits * ROWS, k0 = part * a.klen, k1 = min(a.k, k0 + a.klen);
    const int id = lora_id<ROWS>(a, r0);
    uint64_t left = __ballot(id >= 0);
    const int odd = lane & 1;
    const T *x[RW][2];   // rows of the lane pair, from its piece of a step on: the even lane's is the first 8 q values, the odd one's 32 values behind
#pragma unroll
    for (int i = 0; i < RW; ++i)
#pragma unroll
        for (int h = 0; h < 2; ++h) x[i][h] = (const T *) a.x + (int64_t) min(r0 + 16 * i + (i16 & ~1) + h, a.m - 1) * a.ldx + 8 * q + 32 * odd;
    for (int turn = 0; left; ++turn) {
        const int ad = __builtin_amdgcn_readlane(id, __builtin_ctzll(left));
        const uint64_t mine = __ballot(id == ad);
        left &= ~mine;
        if (turn % gridDim.z != blockIdx.z) continue;
        for (int rb = 0; rb < a.r; rb += 16 * RT) {
            const T *A[RT][2];
#pragma unroll
            for (int j = 0; j < RT; ++j)
#pragma unroll
                for (int h = 0; h < 2; ++h) A[j][h] = (const T *) a.A + ((int64_t) ad * a.r + min(rb + 16 * j + (i16 & ~1) + h, a.r - 1)) * a.k + 8 * q + 32 * odd;
            f4 acc[RW][RT] = {};
            int kk = __builtin_amdgcn_readfirstlane(k0 + 64 * wave);
            // whole steps, two sets of operands in turns: the loads ask no condition (the last step's are its own again), so that the
            // compiler counts those in flight and products wait for their own operands only
            const int last = k1 - kk >= 64 ? kk + (k1 - kk - 64) / STEP * STEP : -1;
            if (last >= 0) {
                LowStep<T, RT, RW> s0, s1;
                s0.load(x, A, kk);
                for (;;) {
                    s1.load(x, A, min(kk + STEP, last));
                    lora_keep_order();
                    s0.swap();
                    s0.add(acc);
                    if ((kk += STEP) > last) break;
                    s0.load(x, A, min(kk + STEP, last));
                    lora_keep_order();
                    s1.swap();
                    s1.add(acc);
                    if ((kk += STEP) > last) break;
                }
            }
            for (; kk < k1; kk += STEP) {   // the lane's own rows, up to the part's end
                LowStep<T, RT, RW> s;
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    const int c = kk + 8 * q + 32 * h;
#pragma unroll
                    for (int i = 0; i < RW; ++i) s.x[i][h] = lora_ld<T, 8>((const T *) a.x + (int64_t) min(r0 + 16 * i + i16, a.m - 1) * a.ldx, c, k1);
#pragma unroll
                    for (int j = 0; j < RT; ++j) s.w[j][h] = lora_ld<T, 8>((const T *) a.A + ((int64_t) ad * a.r + min(rb + 16 * j + i16, a.r - 1)) * a.k, c, k1);
                }
                s.add(acc);
            }
#pragma unroll
            for (int i = 0; i < RW; ++i) {
                if (!(mine >> (16 * i) & 0xffff)) continue;   // (the same in every wave)
#pragma unroll
                for (int j = 0; j < RT; ++j) *(f4 *) &s_acc[wave][i16][16 * j + 4 * q] = acc[i][j];
                __syncthreads();
                for (int e = threadIdx.x; e < 16 * 16 * RT; e += 256) {
                    const int row = e / (16 * RT), c = e % (16 * RT);
                    if ((mine >> (16 * i + row) & 1) && rb + c < a.r)
                        a.low[((int64_t) part * a.m + r0 + 16 * i + row) * a.r + rb + c] = (s_acc[0][row][c] + s_acc[1][row][c]) + (s_acc[2][row][c] + s_acc[3][row][c]);
                }
                __syncthreads();
            }
        }
    }
}

// the sums over the parts of N low products from rank c on (those below r)
template <int N> __device__ __forceinline__ void lora_sum(const float *low, int64_t between, int splits, int c, int r, float (&v)[N]) {
#pragma unroll
    for (int i = 0; i < N; ++i) v[i] = 0.0f;
    if (c >= r) return;
    constexpr int U = N >= 16 ? 2 : N >= 8 ? 4 : 8, P = N < 4 ? N : 4;   // parts on their way together
    for (int sp = 0; sp < splits; sp += U) {
        typename LoraVec<float, P>::vec p[U][N / P];
#pragma unroll
        for (int h = 0; h < U; ++h)
#pragma unroll
            for (int i = 0; i < N / P; ++i) p[h][i] = lora_ld<float, P>(low + (int64_t) min(sp + h, splits - 1) * between, c + P * i, r);
#pragma unroll
        for (int h = 0; h < U; ++h)
            if (sp + h < splits) {
#pragma unroll
                for (int i = 0; i < N; ++i) v[i] += p[h][i / P][i % P];
            }
    }
}

// The second product and the epilogue: 16 RT rows x 64 columns a wave and item; the block's four waves have the same rows, whose
// low products they keep in LDS as the matrix instructions' operands.  Column tile j's operand row i is column 16 j + i for fp32
// outputs and 32 (j / 2) + 8 (i / 4) + 4 (j % 2) + i % 4 for 16-bit ones, so that a lane holds 16-byte pieces of its row.  A turn of 64
// columns is an item for each of the rows' adapters: its columns of B, its rows' residual, products, outputs (a row tile where
// prompts meet is multiplied for each).  Up to rank 64 the next item's loads are on their way while an item is worked on.
// KK: ranks in units of 32.  KIND: UP_WHOLE where n and r are multiples of 8 and there is a resid: pieces then lie inside or outside as a
// whole, loads ask no condition and outside ones are clamped (with conditions 4096 rows, 4096 -> 7168, rank 64, both launches: 89 us
// for 66); UP_ALONE the same without a resid (68 us by UP_ANY, 50 so); UP_ANY else.
enum { UP_ANY, UP_WHOLE, UP_ALONE };
template <typename T, typename O, int RT, int KK, int KIND> struct UpItem {
    static constexpr bool WHOLE = KIND != UP_ANY;
    static constexpr int PN = 16 / sizeof(O), NP = 16 / PN, LOADS = 4 * KK + (KIND == UP_ALONE ? 0 : RT * NP);   // values of a piece, a lane's pieces of a row, loads
    typedef typename LoraVec<O, PN>::vec PT;
    v8<T> b[KK][4];
    PT res[RT][NP];
    uint64_t mine, write;   // the item's rows that have its adapter, and all that it writes
    int c0;

    // piece p belongs to the lane pair's even row (p % 2 = 0) or odd row: even lanes have the columns of pieces 2 (p / 2), odd ones those of the next
    __device__ __forceinline__ static int row_of(int i, int p, int lane) { return 16 * i + (lane & 14) + (p & 1); }
    __device__ __forceinline__ int col_of(int p, int lane) const { return c0 + (2 * (p >> 1) + (lane & 1)) * 4 * PN + PN * (lane >> 4); }
    __device__ __forceinline__ void load(const LoraArgs &a, int ad, const char *rbase, uint32_t ldr, int lane) {
        const int q = lane >> 4, i16 = lane & 15;
        // ranks behind the last are other ranks (WHOLE: taken out piece by piece at their use) or the next rows' values (taken out by mask());
        // at the end of all matrices there are none
        const int64_t base = (int64_t) max(ad, 0) * a.n * a.r;
        const bool inside = WHOLE || base + (int64_t) min(c0 + 63, a.n - 1) * a.r + 32 * KK <= (int64_t) a.n_local * a.n * a.r;   // (the same in every lane)
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const int c = min(c0 + (PN == 4 ? 16 * j + i16 : 32 * (j >> 1) + 8 * (i16 >> 2) + 4 * (j & 1) + (i16 & 3)), a.n - 1);
            const T *B = (const T *) a.B + base + (int64_t) c * a.r;
#pragma unroll
            for (int h = 0; h < KK; ++h) {
                const int at = 32 * h + 8 * q;
                if (WHOLE) b[h][j] = lora_get<T, 8>(B + min(at, a.r - 8));
                else if (inside) b[h][j] = lora_get<T, 8>(B + at);
                else b[h][j] = lora_ld<T, 8>(B, at, a.r);
            }
        }
        const int first = __builtin_ctzll(write);
        auto at = [&](int i, int p) {   // a row that is not to be written: one that is, as for other lanes
            const uint32_t row = write >> row_of(i, p, lane) & 1 ? row_of(i, p, lane) : first;
            return row * ldr;
        };
#pragma unroll
        for (int i = 0; i < RT; ++i)
#pragma unroll
            for (int p = 0; p < NP; ++p) {
                if (KIND == UP_ALONE) res[i][p] = PT{};
                else if (WHOLE) res[i][p] = lora_get<O, PN>((const O *) (rbase + (at(i, p) + min(col_of(p, lane), a.n - PN) * (uint32_t) sizeof(O))));
                else res[i][p] = a.resid ? lora_ld<O, PN>((const O *) (rbase + at(i, p)), col_of(p, lane), a.n) : PT{};
            }
    }
    __device__ __forceinline__ void mask(int r, int q) {
        typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
#pragma unroll
        for (int h = 0; h < KK; ++h) {
            const int n = r - 32 * h - 8 * q;   // values of the piece that are the row's
            u32x4 m;
#pragma unroll
            for (int i = 0; i < 4; ++i) m[i] = n >= 2 * i + 2 ? 0xffffffffu : n == 2 * i + 1 ? 0xffffu : 0u;
#pragma unroll
            for (int j = 0; j < 4; ++j) b[h][j] = __builtin_bit_cast(v8<T>, __builtin_bit_cast(u32x4, b[h][j]) & m);
        }
    }
};
template <typename T, typename O, int RT, int KK, int KIND> __global__ __launch_bounds__(256) void k_lora_up(const LoraArgs a, int gy) {
    typedef UpItem<T, O, RT, KK, KIND> Item;
    constexpr bool WHOLE = Item::WHOLE;
    constexpr int R = 32 * KK, LD = R + 8, ROWS = 16 * RT, PN = Item::PN, NP = Item::NP;
    constexpr int PARTS = sizeof(O) == 4 ? 3 : 2;   // 16-bit values of a low product
    __shared__ __attribute__((aligned(16))) T s_low[PARTS][ROWS * LD];
    __shared__ float s_scale[ROWS];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), q = lane >> 4, i16 = lane & 15;
    const int blk = xcd_tile(blockIdx.x, gridDim.x);   // neighbouring tiles on one XCD: they share adapters
    const int r0 = blk / gy * ROWS;
    const int id = lora_id<ROWS>(a, r0);
    // the adapters of the tile that are this block's: their rows
    uint64_t left = __ballot(id >= 0), rows = 0;
    for (int turn = 0; left; ++turn) {
        const uint64_t mine = __ballot(id == __builtin_amdgcn_readlane(id, __builtin_ctzll(left)));
        left &= ~mine;
        if (turn % gridDim.z == blockIdx.z) rows |= mine;
    }
    // rows without an adapter are the first blocks'
    uint64_t none = __ballot(id < 0 && lane < ROWS && r0 + lane < a.m);
    if (blockIdx.z || (a.resid == a.out && a.ldr == a.ldo)) none = 0;
    if (!(rows | none)) return;   // (the same in every wave)
    // the tile's rows by 32-bit offsets (rows of at most 2^24 bytes)
    const char *rbase = (const char *) a.resid + (int64_t) r0 * a.ldr * (int) sizeof(O);
    char *obase = (char *) a.out + (int64_t) r0 * a.ldo * (int) sizeof(O);
    const uint32_t ldr = (uint32_t) a.ldr * (uint32_t) sizeof(O), ldo = (uint32_t) a.ldo * (uint32_t) sizeof(O);
    int c0 = (blk % gy * 4 + wave) * 64;
    left = rows;   // those of the turn's items that are still to come
    auto next = [&](Item &s) {   // the next item's loads
        const int ad = left ? __builtin_amdgcn_readlane(id, __builtin_ctzll(left)) : -1;
        s.mine = left ? __ballot(id == ad) : 0;
        s.write = s.mine | (left == rows ? none : 0);   // with the first of a turn those without an adapter
        s.c0 = min(c0, a.n - 1);
        s.load(a, ad, rbase, ldr, lane);
        left &= ~s.mine;
        if (!left) { left = rows; c0 += gy * 256; }
    };
    Item s0, s1;
    next(s0);   // on its way while the low products are added up
    // TPR threads a row with PER neighbouring ranks each
    constexpr int TPR = 256 / ROWS, PER = R / TPR;
    if (rows) {
        const int row = threadIdx.x / TPR, t = threadIdx.x % TPR;
        float v[PER], top = 0.0f;
        const float *low = a.low + (int64_t) (r0 + row) * a.r;
        const int64_t between = (int64_t) a.m * a.r;
        const int end = rows >> row & 1 ? a.r : 0;
        lora_sum<PER>(low, between, a.splits, t * PER, end, v);
        float up = 1.0f;
        if constexpr (__is_same(T, f16)) {
#pragma unroll
            for (int i = 0; i < PER; ++i) top = fmaxf(top, fabsf(v[i]));
#pragma unroll
            for (int o = 1; o < TPR; o <<= 1) top = fmaxf(top, __shfl_xor(top, o));
            const int e = (int) (__float_as_uint(top) >> 23) - 127;   // 2^e <= top
            if (top < __builtin_huge_valf() && e > -100) up = __uint_as_float((uint32_t) (127 + min(max(13 - e, -113), 113)) << 23);   // the largest to 2^13 .. 2^14
        }
        if (t == 0) {
            const int my = end ? a.ids[r0 + row] : 0;
            s_scale[row] = (a.scale && end ? a.scale[my] : 1.0f) * (1.0f / up);
        }
        constexpr int P = PER < 8 ? PER : 8;
        typedef T vt __attribute__((ext_vector_type(P)));
#pragma unroll
        for (int g = 0; g < PER; g += P) {
            vt part[PARTS];
#pragma unroll
            for (int i = 0; i < P; ++i) {
                float rest = v[g + i] * up;
                part[0][i] = (T) rest;
#pragma unroll
                for (int h = 1; h < PARTS; ++h) {
                    rest -= (float) part[h - 1][i];
                    rest = rest - rest == 0.0f ? rest : 0.0f;   // (none of an infinity)
                    part[h][i] = (T) rest;
                }
            }
#pragma unroll
            for (int h = 0; h < PARTS; ++h) *(vt *) &s_low[h][row * LD + t * PER + g] = part[h];
        }
    }
    __syncthreads();
    auto work = [&](Item &s) {
        if (!WHOLE && a.r < R) s.mask(a.r, q);
#pragma unroll
        for (int i = 0; i < RT; ++i) {
            if (!(s.write >> (16 * i) & 0xffff)) continue;
            const int r = 16 * i + i16;
            f4 acc[4] = {};
            if (s.mine >> (16 * i) & 0xffff) {
#pragma unroll
                for (int h = 0; h < KK; ++h) {
                    v8<T> low[PARTS];
#pragma unroll
                    for (int e = 0; e < PARTS; ++e) low[e] = *(const v8<T> *) &s_low[e][r * LD + 32 * h + 8 * q];
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        const v8<T> w = !WHOLE || 32 * h + 8 * q < a.r ? s.b[h][j] : v8<T>{};
#pragma unroll
                        for (int e = PARTS - 1; e >= 0; --e) acc[j] = mfma16(w, low[e], acc[j]);   // the smallest first
                    }
                }
            }
            const bool has = s.mine >> r & 1;
            const float sc = has ? s_scale[r] : 0.0f;
#pragma unroll
            for (int j = 0; j < 4; ++j)
#pragma unroll
                for (int e = 0; e < 4; ++e) acc[j][e] = has ? acc[j][e] * sc : 0.0f;   // (nothing of other adapters' values)
#pragma unroll
            for (int p = 0; p < NP; p += 2) {
                // the pair's pieces change places: those of piece p and p + 1 become the even row's and the odd row's
#pragma unroll
                for (int e = 0; e < PN / 4; ++e) pair_swap(acc[p * (PN / 4) + e], acc[(p + 1) * (PN / 4) + e]);
#pragma unroll
                for (int o = p; o < p + 2; ++o) {
                    typename LoraVec<O, PN>::type v;
#pragma unroll
                    for (int e = 0; e < PN; ++e) v[e] = (O) (acc[o * (PN / 4) + (e >> 2)][e & 3] + (float) s.res[i][o][e]);
                    const int row = Item::row_of(i, o, lane), c = s.col_of(o, lane);
                    if (!(s.write >> row & 1) || c >= a.n) continue;
                    O *to = (O *) (obase + ((uint32_t) row * ldo + (uint32_t) c * (uint32_t) sizeof(O)));
                    if (WHOLE || c + PN <= a.n) *(typename LoraVec<O, PN>::type *) to = v;
                    else {
#pragma unroll
                        for (int e = 0; e < PN; ++e) if (c + e < a.n) to[e] = v[e];
                    }
                }
            }
        }
    };
    // the item's own loads have come when only the next one's are out (told to the compiler here: behind stores that only some lanes
    // make it could not count, and would wait for the next item's loads as well)
    auto arrived = [] {
        constexpr int L = Item::LOADS;
        lora_keep_order();
        __builtin_amdgcn_s_waitcnt((L & 15) | 0x0F70 | (L >> 4 & 3) << 14);
        lora_keep_order();
    };
    if ((blk % gy * 4 + wave) * 64 >= a.n) return;
    if constexpr (KK <= 2) {
        for (;;) {
            if (c0 >= a.n) { work(s0); break; }   // (the last item)
            next(s1);
            arrived();
            work(s0);
            if (c0 >= a.n) { work(s1); break; }
            next(s0);
            arrived();
            work(s1);
        }
    } else {   // (two items of high rank do not fit the registers)
        for (;;) {
            work(s0);
            if (c0 >= a.n) break;
            next(s0);
        }
    }
}

// Few rows: tiles of 16, a part of the contraction for each 256 values begun at most.  Many: tiles of 32, a part for each 1024 begun (the
// second launch reads every part again).  Parts are multiples of 256 values and the last has what is left, which may be one.
// As many parts as make 512 blocks, or 384 of many rows: tiles where prompts meet have more blocks, which would start a second round (4096 rows of 24 prompts, rank 64: 3 parts for 4, 59.9 us for 62.8; 2048 rows of 12, k 7168, 30.5 for 34).
constexpr int LORA_MANY = 256;
LoraCut lora_cut(int m, int k) {
    const bool many = m >= LORA_MANY;
    const int rows = many ? 32 : 16, least = many ? 1024 : 256;
    const int tiles = (m + rows - 1) / rows, most = std::max(1, std::min(32, (k + least - 1) / least));
    const int want = std::max(1, std::min(most, ((many ? 384 : 512) + tiles - 1) / std::max(1, tiles)));
    const int klen = ((k + want - 1) / want + 255) / 256 * 256;
    return LoraCut{(int) (((int64_t) k + klen - 1) / klen), klen};
}

// how many of a tile's adapters go side by side, in blocks of their own, up to `most` blocks in all (a tile of one adapter leaves the
// others empty)
static uint32_t lora_deal(int64_t blocks, int most) { return (uint32_t) std::max<int64_t>(1, std::min<int64_t>(16, most / std::max<int64_t>(1, blocks))); }

template <typename T, typename O> static int launch_up(const LoraArgs &a, hipStream_t s) {
    const bool whole = a.n % 8 == 0 && a.r % 8 == 0, tall = a.r <= 64 && a.m >= LORA_MANY;
    constexpr int TALL = sizeof(O) == 4 ? 2 : 4;   // row tiles whose residual fits the registers twice
    const int tiles = tall ? (a.m + 16 * TALL - 1) / (16 * TALL) : (a.m + 15) / 16, cols = (a.n + 255) / 256;
    // many rows: about two blocks a CU, that take several turns with their rows' low products
    const int turns = std::max(1, (int) (((int64_t) tiles * cols + 511) / 512)), gy = (cols + turns - 1) / turns;
    const dim3 up(tiles * gy, 1, lora_deal((int64_t) tiles * gy, tall ? 512 : 1024));
#define HY_UP(RT, KK) { if (!whole) k_lora_up<T, O, RT, KK, UP_ANY><<<up, 256, 0, s>>>(a, gy); else if (a.resid) k_lora_up<T, O, RT, KK, UP_WHOLE><<<up, 256, 0, s>>>(a, gy); \
                       else k_lora_up<T, O, RT, KK, UP_ALONE><<<up, 256, 0, s>>>(a, gy); }
    if (a.r <= 32) { if (tall) HY_UP(TALL, 1) else HY_UP(1, 1) }
    else if (a.r <= 64) { if (tall) HY_UP(TALL, 2) else HY_UP(1, 2) }
    else if (a.r <= 128) HY_UP(1, 4)
    else HY_UP(1, 8)
#undef HY_UP
    return check_launch("hy_lora");
}
template <typename T> static int launch_lora_t(const LoraArgs &a, hipStream_t s) {
    const bool many = a.m >= LORA_MANY;
    const int tiles = (a.m + (many ? 31 : 15)) / (many ? 32 : 16);
    const dim3 low(tiles * a.splits, 1, lora_deal((int64_t) tiles * a.splits, many ? 2048 : 1024));
#define HY_LOW(RT) { if (many) k_lora_low<T, RT, 2><<<low, 256, 0, s>>>(a); else k_lora_low<T, RT, 1><<<low, 256, 0, s>>>(a); }
    if (a.r <= 16) HY_LOW(1) else if (a.r <= 32) HY_LOW(2) else HY_LOW(4)
#undef HY_LOW
    if (const int rc = check_launch("hy_lora")) return rc;
    return a.out_f32 ? launch_up<T, float>(a, s) : launch_up<T, T>(a, s);
}
int launch_lora(int type, const LoraArgs &a, hipStream_t s) { return type == HY_BF16 ? launch_lora_t<bf16>(a, s) : launch_lora_t<f16>(a, s); }

} // namespace hy
