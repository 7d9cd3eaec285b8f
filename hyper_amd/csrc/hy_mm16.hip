// 16-bit matrix products for every shape, stride and alignment: 64 x 64 output tiles staged one element at a time.
#include "hy_mm16.cuh"

#include <algorithm>

namespace hy {

// One 64 x 64 tile a block of four waves (32 x 32 each), contraction steps of 32 through LDS rows of [row or column][k].
// Elements are loaded one at a time with their own bounds, zeros outside, so any size, stride and 2-byte alignment will do.
template <typename T, int KIND, bool DUAL> __global__ __launch_bounds__(256) void k_mm_any(const MMArgs a) {
    constexpr int BK = 32, LD = BK + 8;
    __shared__ __attribute__((aligned(16))) T s_p[64 * LD], s_q[64 * LD];
    __shared__ int s_row[64], s_pair[64];
    __shared__ float s_db[32][64];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, wc = wave & 1, wr = wave >> 1;
    constexpr int BN = DUAL ? 32 : 64;
    const int ncol = (a.N + BN - 1) / BN;
    Group g;
    int tile, col;
    if constexpr (KIND == TN) {
        g = find_expert<256>(a, blockIdx.y);
        tile = blockIdx.x / ncol;
        col = blockIdx.x % ncol;
    } else {
        int part;
        if (!find_tile<256, 64>(a, ncol, false, g, tile, col, part)) return;
    }
    const int c0 = col * BN, r0 = tile * 64;
    if constexpr (KIND != TN) {
        if (tid < 64) {
            const int p = r0 + tid < g.cnt ? pair_of(a, g, r0 + tid) : -1;
            s_pair[tid] = p;
            s_row[tid] = p < 0 ? -1 : div_k(p, a.kq);
        }
        __syncthreads();
    }
    f4 acc[2][2] = {};
    float db[8] = {};
    const int K = KIND == TN ? g.cnt : a.K;
    for (int part = 0; part < (KIND == NN && a.P2 ? 2 : 1); ++part) {
        const T *P = (const T *) (part ? a.P2 : a.P) + (KIND == TN ? 0 : (int64_t) g.le * a.pstride);
        const T *P2 = DUAL ? (const T *) a.P2 + (int64_t) g.le * a.pstride : nullptr;
        const T *Q = (const T *) (part ? a.Q2 : a.Q);
        for (int k0 = 0; k0 < K; k0 += BK) {
            T pv[8], qv[8];
            if constexpr (KIND == TN) {
                const int kk = k0 + (tid >> 3), p = kk < K ? pair_of_expert(a, g, kk) : -1;
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    const int r = r0 + (tid & 7) * 8 + i, c = c0 + (tid & 7) * 8 + i;
                    qv[i] = p >= 0 && r < a.R ? Q[(int64_t) div_k(p, a.kq) * a.ldq + r] : (T) 0.0f;
                    pv[i] = p >= 0 && c < a.N ? P[(int64_t) div_k(p, a.kp) * a.ldp + c] : (T) 0.0f;
                    db[i] += (float) qv[i];
                }
            } else {
                const int row = s_row[tid >> 2];
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    const int kk = k0 + (tid & 3) * 8 + i;
                    qv[i] = row >= 0 && kk < K ? Q[(int64_t) row * a.ldq + kk] : (T) 0.0f;
                }
                if constexpr (KIND == NN) {
                    const int kk = k0 + (tid >> 3);
#pragma unroll
                    for (int i = 0; i < 8; ++i) {
                        const int c = c0 + (tid & 7) * 8 + i;
                        pv[i] = kk < K && c < a.N ? P[(int64_t) kk * a.ldp + c] : (T) 0.0f;
                    }
                } else {
                    const int j = tid >> 2;   // tile column; gated: 16 gate columns, then the same 16 of up
                    const int c = DUAL ? c0 + (j >> 5) * 16 + (j & 15) : c0 + j;
                    const T *M = DUAL && (j & 16) ? P2 : P;
#pragma unroll
                    for (int i = 0; i < 8; ++i) {
                        const int kk = k0 + (tid & 3) * 8 + i;
                        pv[i] = kk < K && c < a.N ? M[(int64_t) c * a.ldp + kk] : (T) 0.0f;
                    }
                }
            }
            __syncthreads();   // the previous step's operands are read
            if constexpr (KIND == TN) {
#pragma unroll
                for (int i = 0; i < 8; ++i) s_q[((tid & 7) * 8 + i) * LD + (tid >> 3)] = qv[i];
            } else {
#pragma unroll
                for (int i = 0; i < 8; ++i) s_q[(tid >> 2) * LD + (tid & 3) * 8 + i] = qv[i];
            }
            if constexpr (KIND == NT) {
#pragma unroll
                for (int i = 0; i < 8; ++i) s_p[(tid >> 2) * LD + (tid & 3) * 8 + i] = pv[i];
            } else {
#pragma unroll
                for (int i = 0; i < 8; ++i) s_p[((tid & 7) * 8 + i) * LD + (tid >> 3)] = pv[i];
            }
            __syncthreads();
            v8<T> fp[2], fq[2];
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                fp[i] = *(const v8<T> *) &s_p[(wc * 32 + i * 16 + (lane & 15)) * LD + (lane >> 4) * 8];
                fq[i] = *(const v8<T> *) &s_q[(wr * 32 + i * 16 + (lane & 15)) * LD + (lane >> 4) * 8];
            }
#pragma unroll
            for (int i = 0; i < 2; ++i)
#pragma unroll
                for (int j = 0; j < 2; ++j) acc[i][j] = mfma16(fp[i], fq[j], acc[i][j]);
        }
    }
#pragma unroll
    for (int j = 0; j < 2; ++j) {
        const int i = wr * 32 + j * 16 + (lane & 15);
        int row;
        int64_t ob = 0;
        float w = 1.0f;
        if constexpr (KIND == TN) {
            row = r0 + i < a.R ? r0 + i : -1;
            ob = (int64_t) blockIdx.y * a.ostride;
        } else {
            row = s_pair[i];
            if (a.wts && row >= 0) w = a.wts[row];
        }
        if (row < 0) continue;
        float v[2][4];
#pragma unroll
        for (int i2 = 0; i2 < 2; ++i2)
#pragma unroll
            for (int e = 0; e < 4; ++e) v[i2][e] = acc[i2][j][e];
        if constexpr (DUAL) epi_glu<T, 4>(a, row, c0 + wc * 16 + 4 * (lane >> 4), v[0], v[1]);
        else
#pragma unroll
            for (int i2 = 0; i2 < 2; ++i2) epi_store<T, 4>(a, ob, row, c0 + wc * 32 + i2 * 16 + 4 * (lane >> 4), v[i2], w);
    }
    if constexpr (KIND == TN) {
        if (a.db && c0 == 0) {
            __syncthreads();
#pragma unroll
            for (int i = 0; i < 8; ++i) s_db[tid >> 3][(tid & 7) * 8 + i] = db[i];
            __syncthreads();
            if (tid < 64 && r0 + tid < a.R) {
                float v = 0.0f;
                for (int k = 0; k < 32; ++k) v += s_db[k][tid];
                a.db[r0 + tid] = a.accumulate ? a.db[r0 + tid] + v : v;
            }
        }
    }
}

template <typename T> static int launch_any(int kind, bool dual, const MMArgs &a, hipStream_t s, const char *what) {
    const int64_t ncol = (a.N + (dual ? 31 : 63)) / (dual ? 32 : 64);
    const int64_t items = kind == TN || !a.egrp ? (a.R + 63) / 64 : (a.n_pairs + 63) / 64 + a.max_active;
    const int64_t blocks = ncol * items;
    if (blocks <= 0) return HY_OK;
    if (const int rc = check_blocks(what, blocks)) return rc;
    const dim3 grid((uint32_t) blocks, kind == TN ? (uint32_t) std::max(1, a.n_local) : 1u);
    if (kind == NT) {
        if (dual) k_mm_any<T, NT, true><<<grid, 256, 0, s>>>(a);
        else k_mm_any<T, NT, false><<<grid, 256, 0, s>>>(a);
    } else if (kind == NN) k_mm_any<T, NN, false><<<grid, 256, 0, s>>>(a);
    else k_mm_any<T, TN, false><<<grid, 256, 0, s>>>(a);
    return check_launch(what);
}

// 16-byte rows: what the tile kernels read in 16-byte pieces starts and repeats on 16 bytes, and no piece passes the end of
// its row
static bool rows16b(const void *p, int64_t ld, int64_t stride, int len) { return ((uintptr_t) p & 15) == 0 && ld % 8 == 0 && stride % 8 == 0 && len % 8 == 0; }

int launch_mm(int kind, int type, bool dual, const MMArgs &a, hipStream_t s, const char *what) {
    const int plen = kind == NT ? a.K : a.N, qlen = kind == TN ? a.R : a.K;
    if (rows16b(a.P, a.ldp, a.pstride, plen) && rows16b(a.P2, a.ldp, a.pstride, plen) && rows16b(a.Q, a.ldq, 0, qlen) && rows16b(a.Q2, a.ldq, 0, qlen)) {
        if (kind == NT) return launch_tiles_nt(type, dual, a, s, what);
        if (kind == NN) return launch_tiles_nn(type, a, s, what);
        return launch_tiles_tn(type, a, s, what);
    }
    return type == HY_BF16 ? launch_any<bf16>(kind, dual, a, s, what) : launch_any<f16>(kind, dual, a, s, what);
}

} // namespace hy
