// The tile kernels of the 16-bit matrix products: operands by LDS DMA, 16 x 16 x 32 matrix instructions.
#pragma once
#include "hy_mm16.cuh"

namespace hy {

// 16 bytes a lane from per-lane addresses to 1 KB of LDS at `lds` (lane l's bytes at lds + 16 l), in flight when it returns
__device__ __forceinline__ void dma16(const char *src, uint32_t lds) {
    uint32_t keep;   // M0 holds the LDS address of a DMA; it is saved and restored around it
    asm volatile("s_mov_b32 %0, m0\n\ts_mov_b32 m0, %2\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, off\n\ts_mov_b32 m0, %0"
                 : "=&s"(keep) : "v"(src), "s"(__builtin_amdgcn_readfirstlane(lds)) : "memory");
}
template <typename V> __device__ __forceinline__ V lds_get(uint32_t addr) { return *(const __attribute__((address_space(3))) V *) (uintptr_t) addr; }
typedef short s4 __attribute__((ext_vector_type(4)));
// transposing read: of each 16 lanes, lane j names 4 values of row j / 4 and gets the four rows' value of column j
__device__ __forceinline__ s4 lds_get_tr(uint32_t addr) {
    return __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s4 *) (uintptr_t) addr);
}
static __device__ __attribute__((aligned(16))) const uint32_t g_zero16[4] = {0, 0, 0, 0};

// How an operand's tile of S rows (or columns) by 64 contraction values lies in LDS, S x 128 bytes, 16-byte pieces:
//  along the contraction (TR false): row r at r * 128, its piece c at c ^ (r & 7) -- a fragment read takes 16 rows' piece c
//  across it (TR true): contraction row k at k * 2 S, its pair of pieces u at u ^ F(k), F = k & 3 | bit 3 of k << 2 -- a
//  transposing read takes 32 bytes of the rows 8 q + 0..3 (or 4..7) of two quarters q at a time, eight different F
template <bool TR, int S, int NW> struct Operand {
    static constexpr int N = S / 8 / NW;   // DMAs a wave and stage
    static_assert(N * 8 * NW == S, "whole DMAs");
    static constexpr int BYTES = S * 128;
    static constexpr int CPR = S / 8, RPI = TR ? 64 / CPR : 8;   // pieces a contraction row, rows a DMA
    const char *p[N];

    // the DMA's contraction row within the stage (TR) / first contraction value of the lane's piece (not TR)
    static __device__ __forceinline__ int krow(int wave, int lane, int i) {
        if constexpr (TR) return (wave * N + i) * RPI + lane / CPR;
        else return ((lane & 7) ^ (lane >> 3)) * 8;
    }
    // the lane's row (not TR) / first column (TR) within the tile
    static __device__ __forceinline__ int at(int wave, int lane, int i) {
        if constexpr (TR) {
            const int k = krow(wave, lane, i), pc = lane % CPR, F = (k & 3) | ((k >> 1) & 4);
            return (((pc >> 1) ^ F) * 2 + (pc & 1)) * 8;
        } else return (wave * N + i) * 8 + (lane >> 3);
    }
    static __device__ __forceinline__ uint32_t dst(uint32_t tile, int wave, int i) { return tile + (uint32_t) (wave * N + i) * 1024; }

    // lane's part of the fragment address: 16 rows / columns from `base` (a multiple of 16) on, contraction half kk of the stage
    static __device__ __forceinline__ uint32_t frag_addr(int lane) {
        if constexpr (TR) {
            const int F = ((lane >> 2) & 3) | ((lane >> 2) & 4);
            return (uint32_t) (((lane >> 4) * 8 + ((lane >> 2) & 3)) * 2 * S + F * 32 + (lane & 3) * 8);
        } else return (uint32_t) ((lane & 15) * 128 + (((lane >> 4) ^ (lane & 7)) * 16));
    }
    template <typename T> static __device__ __forceinline__ v8<T> frag(uint32_t tile, uint32_t fa, int base, int kk) {
        if constexpr (TR) {
            const uint32_t ad = tile + (fa ^ (uint32_t) (base * 2)) + (uint32_t) (kk * 64 * S);
            union { s4 h[2]; v8<T> v; } r;
            r.h[0] = lds_get_tr(ad);
            r.h[1] = lds_get_tr(ad + 8 * S);
            return r.v;
        } else return lds_get<v8<T>>(tile + (fa ^ (uint32_t) (kk * 64)) + (uint32_t) (base * 128));
    }
};

// One BM x BN tile (output rows x columns) a block of WP x WQ waves, BN / WP columns by BM / WQ rows each; stages of 64
// contraction values, NST of them in LDS.
template <typename T, int KIND, bool DUAL, int BM, int BN, int WP, int WQ, int NST>
__global__ __launch_bounds__(64 * WP * WQ, 2) void k_mm(const MMArgs a) {
    constexpr int NW = WP * WQ, NTH = 64 * NW, FP = BN / WP / 16, FQ = BM / WQ / 16;
    using OP = Operand<KIND != NT, BN, NW>;
    using OQ = Operand<KIND == TN, BM, NW>;
    constexpr int NDMA = OP::N + OQ::N, STAGE = OP::BYTES + OQ::BYTES;
    __shared__ __attribute__((aligned(1024))) uint8_t s_mem[NST * STAGE];
    __shared__ int s_pair[BM];
    const int tid = threadIdx.x, wave = __builtin_amdgcn_readfirstlane(tid >> 6), lane = tid & 63, wp = wave % WP, wq = wave / WP;
    constexpr int CN = DUAL ? BN / 2 : BN;   // output columns a tile
    const int ncol = (a.N + CN - 1) / CN;
    Group g;
    int tile, col = 0;
    if constexpr (KIND == TN) {
        tile = place_tile<4>(blockIdx.x, (a.R + BM - 1) / BM, ncol, col);
        g = find_expert<NTH>(a, blockIdx.y);
    } else {
        if (!find_item<NTH, BM>(a, [&](int items) { return place_tile<4>(blockIdx.x, items, ncol, col); }, g, tile)) return;
    }
    const int c0 = col * CN, r0 = tile * BM;
    const uint64_t mq = div_magic(a.kq), mp = div_magic(a.kp);
    const int64_t ldp2 = a.ldp * 2, ldq2 = a.ldq * 2;
    OP P;
    OQ Q;
    const char *Pb = (const char *) a.P + (KIND == TN ? 0 : (int64_t) g.le * a.pstride * 2);
    if constexpr (KIND != TN) {
        for (int i = tid; i < BM; i += NTH) s_pair[i] = r0 + i < g.cnt ? pair_of(a, g, r0 + i) : -1;
        __syncthreads();
    }
    const int K = KIND == TN ? g.cnt : a.K;
    // rows and columns outside the matrices read their first one instead (never stored); the contraction's end reads zeros
#pragma unroll
    for (int i = 0; i < OP::N; ++i) {
        const int at = OP::at(wave, lane, i);
        if constexpr (KIND == NT) {
            int c = DUAL ? c0 + (at >> 5) * 16 + (at & 15) : c0 + at;   // gated: 16 gate columns, then the same 16 of up
            if (c >= a.N) c = c0;
            const char *M = DUAL && (at & 16) ? (const char *) a.P2 + (int64_t) g.le * a.pstride * 2 : Pb;
            P.p[i] = M + c * ldp2 + OP::krow(wave, lane, i) * 2;
        } else {
            const int c = c0 + at < a.N ? c0 + at : c0;
            P.p[i] = Pb + c * 2 + (KIND == NN ? OP::krow(wave, lane, i) * ldp2 : 0);
        }
    }
#pragma unroll
    for (int i = 0; i < OQ::N; ++i) {
        const int at = OQ::at(wave, lane, i);
        if constexpr (KIND == TN) {
            const int r = r0 + at < a.R ? r0 + at : r0;
            Q.p[i] = (const char *) a.Q + r * 2;
        } else {
            const int p = max(s_pair[at], 0);
            Q.p[i] = (const char *) a.Q + div_k(p, a.kq, mq) * ldq2 + OQ::krow(wave, lane, i) * 2;
        }
    }
    const uint32_t lds0 = lds_addr(s_mem);
    const int per_part = (K + 63) >> 6, nstage = KIND == NN && a.P2 ? 2 * per_part : per_part;
    const char *zero = (const char *) g_zero16;

    // TN: the pairs of the wave's contraction rows, one stage ahead of their DMAs
    int ip[KIND == TN ? OP::N : 1], iq[KIND == TN ? OQ::N : 1];
    auto look_up = [&](int s) {
        if constexpr (KIND == TN) {
#pragma unroll
            for (int i = 0; i < OP::N; ++i) { const int k = s * 64 + OP::krow(wave, lane, i); ip[i] = k < K ? pair_of(a, g, k) : -1; }
#pragma unroll
            for (int i = 0; i < OQ::N; ++i) { const int k = s * 64 + OQ::krow(wave, lane, i); iq[i] = k < K ? pair_of(a, g, k) : -1; }
        }
    };
    auto issue = [&](int s, int buf) {
        const uint32_t tp = lds0 + (uint32_t) buf * STAGE, tq = tp + OP::BYTES;
        if constexpr (KIND == TN) {
#pragma unroll
            for (int i = 0; i < OP::N; ++i) dma16(ip[i] >= 0 ? P.p[i] + div_k(ip[i], a.kp, mp) * ldp2 : zero, OP::dst(tp, wave, i));
#pragma unroll
            for (int i = 0; i < OQ::N; ++i) dma16(iq[i] >= 0 ? Q.p[i] + div_k(iq[i], a.kq, mq) * ldq2 : zero, OQ::dst(tq, wave, i));
        } else {
            int64_t dp = 0, dq = 0;
            int sl = s;
            if (KIND == NN && s >= per_part) {   // the second part's matrices
                sl = s - per_part;
                dp = (const char *) a.P2 - (const char *) a.P;
                dq = (const char *) a.Q2 - (const char *) a.Q;
            }
            dp += (KIND == NT ? 128 : 64 * ldp2) * (int64_t) sl;
            dq += 128 * (int64_t) sl;
            const bool full = sl * 64 + 64 <= K;
#pragma unroll
            for (int i = 0; i < OP::N; ++i) {
                const char *src = P.p[i] + dp;
                if (!full && sl * 64 + OP::krow(wave, lane, i) >= K) src = zero;
                dma16(src, OP::dst(tp, wave, i));
            }
#pragma unroll
            for (int i = 0; i < OQ::N; ++i) {
                const char *src = Q.p[i] + dq;
                if (!full && sl * 64 + OQ::krow(wave, lane, i) >= K) src = zero;
                dma16(src, OQ::dst(tq, wave, i));
            }
        }
    };

    f4 acc[FP][FQ] = {};
    f4 dbs[KIND == TN ? FQ : 1] = {};
    const bool do_db = KIND == TN && a.db && col == 0 && wp == 0;
    const uint32_t fap = OP::frag_addr(lane), faq = OQ::frag_addr(lane);
    look_up(0);
    for (int s = 0; s < NST - 1; ++s)
        if (s < nstage) { issue(s, s); look_up(s + 1); }
    int buf = 0;
    for (int s = 0; s < nstage; ++s) {
        // this stage has landed for every wave, and every wave is done with the one before
        if (NST > 2 && KIND != TN && s + NST - 2 < nstage) wait_vm<(NST - 2) * NDMA>();
        else wait_vm<0>();
        lds_barrier();
        if (s + NST - 1 < nstage) { issue(s + NST - 1, buf == 0 ? NST - 1 : buf - 1); look_up(s + NST); }
        const uint32_t tp = lds0 + (uint32_t) buf * STAGE, tq = tp + OP::BYTES;
#pragma unroll
        for (int kk = 0; kk < 2; ++kk) {
            v8<T> fp[FP], fq[FQ];
#pragma unroll
            for (int j = 0; j < FQ; ++j) fq[j] = OQ::template frag<T>(tq, faq, wq * (BM / WQ) + j * 16, kk);
#pragma unroll
            for (int i = 0; i < FP; ++i) fp[i] = OP::template frag<T>(tp, fap, wp * (BN / WP) + i * 16, kk);
#pragma unroll
            for (int i = 0; i < FP; ++i)
#pragma unroll
                for (int j = 0; j < FQ; ++j) acc[i][j] = mfma16(fp[i], fq[j], acc[i][j]);
            if constexpr (KIND == TN) {
                if (do_db) {   // the rows' sums as a product with ones
                    v8<T> one;
#pragma unroll
                    for (int e = 0; e < 8; ++e) one[e] = (T) 1.0f;
#pragma unroll
                    for (int j = 0; j < FQ; ++j) dbs[j] = mfma16(one, fq[j], dbs[j]);
                }
            }
        }
        buf = buf == NST - 1 ? 0 : buf + 1;
    }

#pragma unroll
    for (int j = 0; j < FQ; ++j) {
        const int i0 = wq * (BM / WQ) + j * 16 + (lane & 15);
        int row;
        int64_t ob = 0;
        float w = 1.0f;
        if constexpr (KIND == TN) {
            row = r0 + i0 < a.R ? r0 + i0 : -1;
            ob = (int64_t) blockIdx.y * a.ostride;
            if (do_db && lane < 16 && row >= 0) a.db[row] = a.accumulate ? a.db[row] + dbs[j][0] : dbs[j][0];
        } else {
            row = s_pair[i0];
            if (a.wts && row >= 0) w = a.wts[row];
        }
        if (row < 0) continue;
        const int cl = c0 + wp * (CN / WP) + 4 * (lane >> 4);
        if constexpr (DUAL) {
#pragma unroll
            for (int i = 0; i < FP; i += 2) epi_glu<T>(a, row, cl + i * 8, acc[i][j], acc[i + 1][j]);
        } else {
#pragma unroll
            for (int i = 0; i < FP; ++i) epi_store<T>(a, ob, row, cl + i * 16, acc[i][j], w);
        }
    }
}

template <typename T, int KIND, bool DUAL, int BM, int BN, int WP, int WQ, int NST>
static int launch_tile(const MMArgs &a, hipStream_t s, const char *what) {
    const int64_t ncol = (a.N + (DUAL ? BN / 2 : BN) - 1) / (DUAL ? BN / 2 : BN);
    const int64_t items = KIND == TN || !a.egrp ? ((int64_t) a.R + BM - 1) / BM : ((int64_t) a.n_pairs + BM - 1) / BM + a.max_active;
    const int64_t blocks = ncol * items;
    if (blocks <= 0) return HY_OK;
    if (blocks > 0x7fffffffll) { set_error("%s: %lld tiles", what, (long long) blocks); return HY_EBAD_SHAPE; }
    k_mm<T, KIND, DUAL, BM, BN, WP, WQ, NST><<<dim3((uint32_t) blocks, KIND == TN && a.egrp ? (uint32_t) a.n_local : 1u), 64 * WP * WQ, 0, s>>>(a);
    return check_launch(what);
}

} // namespace hy
