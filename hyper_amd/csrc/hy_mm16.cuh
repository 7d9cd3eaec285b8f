// 16-bit (bf16 / fp16) matrix products with fp32 sums: what the kernels share.
//
// One description covers the linear layer, the products grouped by expert and their gradients.  An output tile has rows
// (operand Q: token or pair rows) and columns (operand P: a weight's rows or columns); KIND says where the contraction lies:
//   NT  out[r][c] = sum_k Q[r][k] P[c][k]      forward: Q = x or h, P = W                (both contiguous along k)
//   NN  out[r][c] = sum_k Q[r][k] P[k][c]      gradient of the rows: Q = dz, P = W
//   TN  out[r][c] = sum_k Q[k][r] P[k][c]      gradient of the weights: Q = dz, P = x, k over the (gathered) rows
// P is the matrix instruction's A operand and Q its B operand: lane l of a 16 x 16 product then holds columns
// 4 (l / 16) .. + 3 of row l % 16, four neighbours of one output row, which it stores together.
#pragma once
#include "hy_div.h"
#include "hy_internal.h"

#include <algorithm>

namespace hy {

enum { NT = 0, NN = 1, TN = 2 };

typedef __bf16 bf16;
typedef _Float16 f16;
typedef float f4 __attribute__((ext_vector_type(4)));
template <typename T> using v8 = T __attribute__((ext_vector_type(8)));
template <typename T> using v4 = T __attribute__((ext_vector_type(4)));

__device__ __forceinline__ f4 mfma16(v8<bf16> a, v8<bf16> b, f4 c) { return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0); }
__device__ __forceinline__ f4 mfma16(v8<f16> a, v8<f16> b, f4 c) { return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0); }

struct MMArgs {
    // operands; P2 / Q2: the second pair of a two-part contraction (NN: up after gate) or the up matrix of a gated product (NT)
    const void *P, *P2, *Q, *Q2;
    int64_t ldp, ldq;        // elements between rows
    int64_t pstride;         // elements between the experts' matrices
    int R, N, K;             // output rows (ungrouped; TN: rows of each gradient), columns, contraction length of one part (TN: ungrouped rows)
    // grouping: pairs order[start ..] of the egrp triples; operand row of pair p is p / kq (TN: also p / kp), output row p
    const int *order, *order_n, *egrp, *slot, *ids;
    int n_local, n_expert, n_pairs, max_active;
    Divisor kq, kp;
    // epilogue: v = acc + bias; z = v; v = act(v) * wts[p] + resid (+ out).  Gated: h = SwiGLU(g, u), g and u on request
    const float *bias, *wts;
    const void *resid;
    void *z, *g, *u, *out;
    int64_t ldr, ldz, ldo, ostride;   // ostride (TN): elements between the experts' gradients
    float *db;                        // TN: sums of Q's columns
    float *part;                      // TN, parts > 1: the sums of each part of the contraction (`parts` of part_len rows), then of db
    int parts, part_len;
    int act, out_f32, accumulate;
    float clamp;
    int bias16;                       // the bias starts on 16 bytes
    int spread;                       // grouped: find_tile's order of tiles
    int split;                        // ungrouped 256 x 256: parts of the tiles that are left for the last turn (1, 2 or 4)
    int vec;                          // out, resid, z, g and u can be moved in 16-byte pieces
};

// Activations in 32 bits: a tile's epilogue evaluates 256 of them a lane, on one wave a SIMD, so the quarter-rate exp2 and
// reciprocal instructions take the place of the correctly rounded forms that the quantized path's contract asks for (a gated
// 256 x 256 tile's epilogue: 26 us with those against 51 us of products).
// exp(x), |x| <= 88: exp2 of the rounded product and the first-order term of its rounding (within 2 units of the last place)
__device__ __forceinline__ float mm_exp(float x) {
    const float t = x * 1.44269502f, lo = fmaf(x, 1.92596299e-8f, fmaf(x, 1.44269502f, -t));
    const float e = __builtin_amdgcn_exp2f(t);
    return fmaf(e, lo * 0.693147182f, e);
}
// 1 / (1 + exp(-x)); 0 below -87.33, where it leaves the normal range
__device__ __forceinline__ float mm_sigmoid(float x) {
    const float r = __builtin_amdgcn_rcpf(1.0f + mm_exp(fminf(fmaxf(-x, -88.0f), 88.0f)));
    return x < -87.33f ? 0.0f : r;
}
// the SwiGLU limit L (0: none) of N gate and up values; NaN is beyond no limit.  (One branch for
// all: as part of each value's expression it ran without a limit too, gate/up of 8192 tokens 597 for 582 us.)
template <int N> __device__ __forceinline__ void mm_limit(float *g, float *u, float L) {
    if (L > 0.0f) {
#pragma unroll
        for (int i = 0; i < N; ++i) { g[i] = g[i] > L ? L : g[i]; u[i] = u[i] > L ? L : u[i] < -L ? -L : u[i]; }
    }
}
__device__ __forceinline__ float mm_swiglu(float g, float u) { return g * mm_sigmoid(g) * u; }
// erfc(|z| / sqrt(2)) and exp(-z^2 / 2) for |z| <= 14 (0 beyond): erfc(a) exp(a^2) is a polynomial in 1 / (1 + a / 2), fitted for
// least relative error on 0 <= a <= 10 (3.5e-7 with its evaluation); the exponent's rounding is carried as in mm_exp
__device__ __forceinline__ void mm_erfc(float z, float &c, float &e) {
    const float x = fminf(fabsf(z), 14.0f);
    const float h = x * x, t = h * -0.721347511f;
    const float lo = fmaf(fmaf(x, x, -h), -0.721347511f, fmaf(h, -9.62981500e-9f, fmaf(h, -0.721347511f, -t)));
    e = __builtin_amdgcn_exp2f(t);
    e = fmaf(e, lo * 0.693147182f, e);
    const float r = __builtin_amdgcn_rcpf(fmaf(x, 0.353553391f, 1.0f));
    float p = -0.0550513342f;
    p = fmaf(p, r, 0.26390329f);
    p = fmaf(p, r, -0.441478103f);
    p = fmaf(p, r, 0.221191511f);
    p = fmaf(p, r, 0.0170772728f);
    p = fmaf(p, r, 0.181250066f);
    p = fmaf(p, r, 0.249793455f);
    p = fmaf(p, r, 0.281098425f);
    p = fmaf(p, r, 0.282221377f);
    p = fmaf(p, r, -6.01127613e-6f);
    c = p * e;
}
__device__ __forceinline__ float mm_act(int act, float z) {
    switch (act) {
    case HY_ACT_RELU: return z > 0.0f || z != z ? z : 0.0f;   // NaN stays NaN
    case HY_ACT_SILU: return z * mm_sigmoid(z);
    case HY_ACT_GELU: {
        float c, e;
        mm_erfc(z, c, e);
        const float h = 0.5f * fminf(z, 14.0f) * c;   // 0 from 14 on, for +inf too; NaN takes the second way out
        return z < 0.0f ? h : z - h;
    }
    case HY_ACT_GELU_TANH: return z * mm_sigmoid(1.5957691216057308f * fmaf(0.044715f * z * z, z, z));
    }
    return z;
}
// act'(z)
__device__ __forceinline__ float mm_act_grad(int act, float z) {
    switch (act) {
    case HY_ACT_RELU: return z > 0.0f ? 1.0f : z != z ? z : 0.0f;
    case HY_ACT_SILU: { const float s = mm_sigmoid(z); return s * fmaf(z, 1.0f - s, 1.0f); }
    case HY_ACT_GELU: {   // Phi(z) + z phi(z)
        float c, e;
        mm_erfc(z, c, e);
        return fmaf(z * 0.39894228040143268f, e, z >= 0.0f ? 1.0f - 0.5f * c : 0.5f * c);
    }
    case HY_ACT_GELU_TANH: {   // z sigmoid(2 a): s + z s (1 - s) 2 a'
        const float s = mm_sigmoid(1.5957691216057308f * fmaf(0.044715f * z * z, z, z));
        const float x = fminf(fmaxf(z, -16.0f), 16.0f);   // s (1 - s) is 0 from there on, while z^2 of large z is infinite
        return fmaf(z * s * (1.0f - s), 1.5957691216057308f * fmaf(0.134145f * x, x, 1.0f), s);
    }
    }
    return 1.0f;
}

// W neighbours (4 or 8) of a T or fp32 matrix, the first n of them; vec: they can be moved in 16-byte pieces
template <typename T, int W> __device__ __forceinline__ void put_n(void *base, int64_t at, const float *v, int n, bool f32, bool vec) {
    if (f32) {
        float *o = (float *) base + at;
        if (vec && n == W) {
#pragma unroll
            for (int i = 0; i < W; i += 4) *(f4 *) (o + i) = f4{v[i], v[i + 1], v[i + 2], v[i + 3]};
        } else {
#pragma unroll
            for (int i = 0; i < W; ++i) if (i < n) o[i] = v[i];
        }
    } else {
        typedef T vt __attribute__((ext_vector_type(W)));
        T *o = (T *) base + at;
        vt t;
#pragma unroll
        for (int i = 0; i < W; ++i) t[i] = (T) v[i];
        if (vec && n == W) *(vt *) o = t;
        else {
#pragma unroll
            for (int i = 0; i < W; ++i) if (i < n) o[i] = t[i];
        }
    }
}
template <typename T, int W> __device__ __forceinline__ void add_n(const void *base, int64_t at, float *v, int n, bool f32, bool vec) {
    if (f32) {
        const float *o = (const float *) base + at;
        if (vec && n == W) {
#pragma unroll
            for (int i = 0; i < W; i += 4) {
                const f4 t = *(const f4 *) (o + i);
#pragma unroll
                for (int j = 0; j < 4; ++j) v[i + j] += t[j];
            }
        } else {
#pragma unroll
            for (int i = 0; i < W; ++i) if (i < n) v[i] += o[i];
        }
    } else {
        typedef T vt __attribute__((ext_vector_type(W)));
        const T *o = (const T *) base + at;
        if (vec && n == W) {
            const vt t = *(const vt *) o;
#pragma unroll
            for (int i = 0; i < W; ++i) v[i] += (float) t[i];
        } else {
#pragma unroll
            for (int i = 0; i < W; ++i) if (i < n) v[i] += (float) o[i];
        }
    }
}
template <int ACT, int W> __device__ __forceinline__ void act_n(float *v) {
#pragma unroll
    for (int i = 0; i < W; ++i) v[i] = mm_act(ACT, v[i]);
}
// outputs c .. c + W - 1 of output row `row` from their sums; ob: element offset of the expert's gradient (TN), w: the pair's weight
template <typename T, int W> __device__ __forceinline__ void epi_store(const MMArgs &a, int64_t ob, int64_t row, int c, float *v, float w) {
    const int n = min(W, a.N - c);
    if (n <= 0) return;
    const bool vec = a.vec;
    if (a.bias) {
#pragma unroll
        for (int i = 0; i < W; ++i) if (i < n) v[i] += a.bias[c + i];
    }
    if (a.z) put_n<T, W>(a.z, row * a.ldz + c, v, n, false, vec);
    switch (a.act) {
    case HY_ACT_RELU: act_n<HY_ACT_RELU, W>(v); break;
    case HY_ACT_SILU: act_n<HY_ACT_SILU, W>(v); break;
    case HY_ACT_GELU: act_n<HY_ACT_GELU, W>(v); break;
    case HY_ACT_GELU_TANH: act_n<HY_ACT_GELU_TANH, W>(v); break;
    }
    if (a.wts) {
#pragma unroll
        for (int i = 0; i < W; ++i) v[i] *= w;
    }
    if (a.resid) add_n<T, W>(a.resid, row * a.ldr + c, v, n, a.out_f32, vec);
    const int64_t at = ob + row * a.ldo + c;
    if (a.accumulate) add_n<T, W>(a.out, at, v, n, a.out_f32, vec);
    put_n<T, W>(a.out, at, v, n, a.out_f32, vec);
}
// gated: h (and g, u) of columns c .. c + W - 1
template <typename T, int W> __device__ __forceinline__ void epi_glu(const MMArgs &a, int64_t row, int c, float *g, float *u) {
    const int n = min(W, a.N - c);
    if (n <= 0) return;
    const int64_t at = row * a.ldo + c;
    if (a.g) { put_n<T, W>(a.g, at, g, n, false, a.vec); put_n<T, W>(a.u, at, u, n, false, a.vec); }
    float h[W];
    mm_limit<W>(g, u, a.clamp);
#pragma unroll
    for (int i = 0; i < W; ++i) h[i] = mm_swiglu(g[i], u[i]);
    put_n<T, W>(a.out, at, h, n, false, a.vec);
}

// ------------------------------------------------------------------ groups

// A block's group: pairs order[start .. start + cnt) (or rows start .. of an ungrouped product) with local expert le
struct Group { int le, start, cnt; };

// triple i of egrp, with every field bounded: a group outside the pairs or without a local expert has no rows
__device__ __forceinline__ Group load_group(const MMArgs &a, int i) {
    const int e = a.egrp[3 * i], start = a.egrp[3 * i + 1], cnt = a.egrp[3 * i + 2];
    Group g{-1, 0, 0};
    if ((uint32_t) e < (uint32_t) a.n_expert && start >= 0 && cnt > 0 && cnt <= a.n_pairs - start) {
        const int s = a.slot[e];
        if ((uint32_t) s < (uint32_t) a.n_local) g = Group{s, start, cnt};
    }
    return g;
}
__device__ __forceinline__ int n_groups(const MMArgs &a) { return max(0, min(a.order_n[1], a.max_active)); }

// The group of this block's work item, found by the whole block of NTH threads: count(i, rows) is the number of items of group i;
// every thread counts those of its few groups and a scan over the block places them.  place(total) says which of the `total`
// items is the block's (below 0: none; the result is false then); `item` becomes its number within the group, gi the group's.
// A group has fewer than 2^24 items (check_blocks).  Groups that overlap, as no hy_moe_order makes them, may have 2^34 in all: the
// scan stops at 2^30, whose last 2^26 no block is placed at, so that at most one thread finds itself named.
template <int NTH, typename C, typename F>
__device__ __forceinline__ bool find_item(const MMArgs &a, C count, F place, Group &g, int &item, int &gi) {
    constexpr int PER = 1024 / NTH;
    static_assert(PER * NTH == 1024, "at most 1024 groups");
    __shared__ int s_w[NTH / 64], s_out[5];
    const int tid = threadIdx.x, lane = tid & 63, ng = n_groups(a);
    Group gs[PER];
    int nt[PER], sum = 0;
#pragma unroll
    for (int j = 0; j < PER; ++j) {
        const int i = tid * PER + j;
        gs[j] = Group{-1, 0, 0};
        if (i < ng) gs[j] = load_group(a, i);
        nt[j] = count(i, gs[j].cnt);
        sum += nt[j];
    }
    auto plus = [](int a, int b) { return (int) min((uint32_t) a + (uint32_t) b, 1u << 30); };
    int inc = sum;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) { const int v = __shfl_up(inc, o); if (lane >= o) inc = plus(inc, v); }
    if (lane == 63) s_w[tid >> 6] = inc;
    if (tid == 0) s_out[2] = 0;
    __syncthreads();
    int pre = inc - sum, all = 0;
#pragma unroll
    for (int w = 0; w < NTH / 64; ++w) { if (w < (tid >> 6)) pre = plus(pre, s_w[w]); all = plus(all, s_w[w]); }
    const int it = place(all);
    if (it < 0) return false;
#pragma unroll
    for (int j = 0; j < PER; ++j) {
        if (it >= pre && it < pre + nt[j]) { s_out[0] = gs[j].le; s_out[1] = gs[j].start; s_out[2] = gs[j].cnt; s_out[3] = it - pre; s_out[4] = tid * PER + j; }
        pre += nt[j];
    }
    __syncthreads();
    g = Group{__builtin_amdgcn_readfirstlane(s_out[0]), __builtin_amdgcn_readfirstlane(s_out[1]), __builtin_amdgcn_readfirstlane(s_out[2])};
    if (!g.cnt) return false;
    item = __builtin_amdgcn_readfirstlane(s_out[3]);
    gi = __builtin_amdgcn_readfirstlane(s_out[4]);
    return true;
}
// The pairs of local matrix `le` (TN), found by the whole block; cnt 0 when it has none.  Start -1: the pairs of several groups
// (experts that share a matrix) one after the other.
template <int NTH> __device__ __forceinline__ Group find_expert(const MMArgs &a, int le) {
    if (!a.egrp) return Group{le, 0, a.K};   // (experts without any pairs: K = 0)
    __shared__ int s_n, s_start, s_cnt;
    if (threadIdx.x == 0) { s_n = 0; s_start = 0; s_cnt = 0; }
    __syncthreads();
    const int ng = n_groups(a);
    for (int i = threadIdx.x; i < ng; i += NTH) {
        const Group g = load_group(a, i);
        if (g.cnt && g.le == le) {
            atomicAdd(&s_n, 1);
            atomicAdd(&s_cnt, g.cnt);
            s_start = g.start;   // (used where one group writes it)
        }
    }
    __syncthreads();
    const int n = __builtin_amdgcn_readfirstlane(s_n), cnt = __builtin_amdgcn_readfirstlane(s_cnt);
    return Group{le, n > 1 ? -1 : __builtin_amdgcn_readfirstlane(s_start), (int) min((uint32_t) cnt, (uint32_t) a.n_pairs)};
}
// pair (or plain row) number i of a group; -1 for an entry outside the pairs
__device__ __forceinline__ int pair_of(const MMArgs &a, const Group &g, int i) {
    if (!a.order) return g.start + i;
    const int p = a.order[g.start + i];
    return (uint32_t) p < (uint32_t) a.n_pairs ? p : -1;
}
// the same of find_expert's group
__device__ __forceinline__ int pair_of_expert(const MMArgs &a, const Group &g, int i) {
    if (!a.order || g.start >= 0) return pair_of(a, g, i);
    const int ng = n_groups(a);
#pragma unroll 1
    for (int j = 0; j < ng; ++j) {
        const Group o = load_group(a, j);
        if (!o.cnt || o.le != g.le) continue;
        if (i < o.cnt) return pair_of(a, o, i);
        i -= o.cnt;
    }
    return -1;
}

// Blocks b, b + 8, .. run on one XCD, whose L2 they share: XCD x gets the tiles from x / 8 of the T tiles on.  -1: no tile.
__device__ __forceinline__ int xcd_tile(uint32_t b, uint32_t T) {
    if (b >= T) return -1;
    const uint32_t q = T >> 3, r = T & 7, x = b & 7;
    return (int) (x * q + min(x, r) + (b >> 3));
}
// The same where a block is alone on its CU and the tiles of an XCD's last, partial turn (of 32) are shared out to S blocks each.
__device__ __forceinline__ int split_tile(uint32_t b, uint32_t T, int S, int &part) {
    const uint32_t q = T >> 3, r = T & 7, x = b & 7, n = q + (x < r), whole = n & ~31u, i = b >> 3;
    const uint32_t at = i < whole ? i : whole + (i - whole) / S;
    part = i < whole ? -1 : (int) ((i - whole) % S);
    return at < n ? (int) (x * q + min(x, r) + at) : -1;
}
inline __host__ int split_parts(int64_t T) {   // what S may be: the parts fit the turn on every XCD
    const int q = (int) (T >> 3) & 31, most = T & 7 ? (q == 31 ? 31 : q + 1) : q;
    return most == 0 || most > 16 ? 1 : most > 8 ? 2 : 4;
}
// tile t of rows x ncol tiles: bands of G row tiles go column by column, so that the blocks that run together read few row and
// few column tiles
template <int G> __device__ __forceinline__ void band_tile(int t, int rows, int ncol, int &tile, int &col) {
    const int band = t / (G * ncol), in = t - band * G * ncol, n = min(G, rows - band * G);
    col = in / n;
    tile = band * G + in % n;
}
// The block's tile of BM rows.  Ungrouped: bands of 4.  Grouped: the groups in order, bands of 8 that do not reach into the next
// group, whose weights are others.  (Groups' ends dealt out behind all whole tiles, to fill the last turn, read the weights
// once more: 64 experts of about 256 rows 160 against 149 us, 128 of about 256 rows 376 against 346.)
// Grouped with few rows a group (spread): the time is the weights' bytes, of which every XCD should fetch as many.  Column tile c
// of group i goes to XCD (i ncol + c) % 8 (tiles dealt out in order instead gave the XCDs of large groups fewer bytes: 288
// experts, 1000 tokens routed by Zipf(1.1): 860 against 785 us).
__device__ __forceinline__ int spread_first(int i, int ncol, int x) { return (x - i * ncol) & 7; }   // XCD x's first column of group i
__device__ __forceinline__ int spread_cols(int i, int ncol, int x) { const int c = spread_first(i, ncol, x); return c < ncol ? (ncol - 1 - c) / 8 + 1 : 0; }
template <int NTH, int BM> __device__ __forceinline__ bool find_tile(const MMArgs &a, int ncol, bool spread, Group &g, int &tile, int &col, int &part) {
    auto tiles = [](int rows) { return (int) (((uint32_t) rows + BM - 1) / BM); };
    const int x = blockIdx.x & 7;
    int gi, t;
    part = -1;
    if (!a.egrp) {
        const uint32_t T = (uint32_t) tiles(a.R) * (uint32_t) ncol;
        if (BM == 256 && a.split > 1) t = split_tile(blockIdx.x, T, a.split, part);
        else t = xcd_tile(blockIdx.x, T);
        if (t < 0) return false;
        g = Group{0, 0, a.R};
        band_tile<4>(t, tiles(a.R), ncol, tile, col);
    } else if (spread) {
        const int it = blockIdx.x >> 3;
        if (!find_item<NTH>(a, [&](int i, int rows) { return tiles(rows) * spread_cols(i, ncol, x); }, [&](int n) { return it < n ? it : -1; }, g, t, gi)) return false;
        band_tile<8>(t, tiles(g.cnt), spread_cols(gi, ncol, x), tile, col);
        col = spread_first(gi, ncol, x) + 8 * col;
    } else {
        if (!find_item<NTH>(a, [&](int, int rows) { return tiles(rows) * ncol; }, [&](int n) { return xcd_tile(blockIdx.x, (uint32_t) n); }, g, t, gi)) return false;
        band_tile<8>(t, tiles(g.cnt), ncol, tile, col);
    }
    return true;
}

// A launch of 2^32 threads or more runs those that 32 bits count and reports nothing: such grids (of blocks of 256) are refused.
inline __host__ int check_blocks(const char *what, int64_t blocks) {
    if (blocks < 1 << 24) return HY_OK;
    set_error("%s: %lld tiles of the output (a call takes less than 2^24)", what, (long long) blocks);
    return HY_EBAD_SHAPE;
}

// launchers (type: HY_F16 / HY_BF16)
int launch_mm(int kind, int type, bool dual, const MMArgs &a, hipStream_t s, const char *what);
int launch_tiles_nt(int type, bool dual, const MMArgs &a, hipStream_t s, const char *what);
int launch_tiles_nn(int type, const MMArgs &a, hipStream_t s, const char *what);
int launch_tiles_tn(int type, const MMArgs &a, hipStream_t s, const char *what);
struct Parts { int n, len; };
Parts dw_parts(int m, int n, int k);   // how the contraction of an n x k gradient of m rows is cut
int launch_mv(int type, bool dual, const MMArgs &a, hipStream_t s, const char *what);
bool few_rows(const MMArgs &a);   // a plain product that launch_few takes
int launch_few(int type, const MMArgs &a, hipStream_t s, const char *what);
int launch_act_bwd(int type, int act, const void *z, int64_t ldz, const void *dy, int64_t lddy, int m, int n, void *dz, int64_t lddz,
                   hipStream_t s);
int launch_swiglu_bwd(int type, const void *g, const void *u, const void *dh, const float *wts, int n_pairs, int ff, float clamp,
                      const int *order, const int *order_n, void *dg, void *du, void *hw, float *dwts, hipStream_t s);
int launch_rows16(int type, const float *x, int64_t xs, int n, int nt, void *out, int64_t ldo, hipStream_t s);

} // namespace hy
