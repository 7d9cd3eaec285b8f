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
// what the wave's lanes wrote to LDS before is what its lanes read behind (LDS operations of a wave keep their order; this
// keeps the compiler's)
__device__ __forceinline__ void wave_sync() {
    asm volatile("" ::: "memory");
    __builtin_amdgcn_wave_barrier();
    asm volatile("" ::: "memory");
}
typedef short s4 __attribute__((ext_vector_type(4)));
// transposing read: of each 16 lanes, lane j names 4 values of row j / 4 and gets the four rows' value of column j
__device__ __forceinline__ s4 lds_get_tr(uint32_t addr) {
    return __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s4 *) (uintptr_t) addr);
}
static __device__ __attribute__((aligned(16))) const uint32_t g_zero16[4] = {0, 0, 0, 0};

// How an operand's tile of S rows (or columns) by BK contraction values lies in LDS, in 16-byte pieces:
//  along the contraction (TR false): row r at r * 2 BK, its piece c at c ^ (r & 7) (BK 64) or c ^ (r >> 2 & 3) (BK 32): a
//  fragment read takes one piece of each of 16 rows, 16 lanes at a time in 16 different places of 256 bytes
//  across it (TR true): contraction row k at k * 2 S, its pair of pieces u at u ^ F(k), F = k & 3 | bit 3 of k << 2: a
//  transposing read takes 32 bytes of the rows 8 q + 0..3 (or 4..7) of two quarters q at a time, eight different F
// Both read at 240 bytes a clock and CU (256 is the most).
template <bool TR, int S, int NW, int BK> struct Operand {
    static constexpr int N = S * BK / 512 / NW;   // DMAs (of 1 KB) a wave and stage
    static_assert(N * 512 * NW == S * BK, "whole DMAs");
    static constexpr int BYTES = S * BK * 2;
    static constexpr int CPR = TR ? S / 8 : BK / 8, RPI = 64 / CPR;   // pieces a stored row, stored rows a DMA
    const char *p[N];

    // the DMA's contraction row within the stage (TR) / first contraction value of the lane's piece (not TR)
    static __device__ __forceinline__ int krow(int wave, int lane, int i) {
        if constexpr (TR) return (wave * N + i) * RPI + lane / CPR;
        else if constexpr (BK == 64) return ((lane & 7) ^ (lane >> 3)) * 8;
        else return ((lane & 3) ^ (lane >> 4)) * 8;
    }
    // the lane's row (not TR) / first column (TR) within the tile
    static __device__ __forceinline__ int at(int wave, int lane, int i) {
        if constexpr (TR) {
            const int k = krow(wave, lane, i), pc = lane % CPR, F = (k & 3) | ((k >> 1) & 4);
            return (((pc >> 1) ^ F) * 2 + (pc & 1)) * 8;
        } else return (wave * N + i) * RPI + lane / CPR;
    }
    static __device__ __forceinline__ uint32_t dst(uint32_t tile, int wave, int i) { return tile + (uint32_t) (wave * N + i) * 1024; }

    // lane's part of the address of a fragment (16 rows / columns from `base`, a multiple of 16, on; 32 contraction values kk)
    static __device__ __forceinline__ uint32_t frag_addr(int lane) {
        if constexpr (TR) {
            const int F = ((lane >> 2) & 3) | ((lane >> 2) & 4);
            return (uint32_t) (((lane >> 4) * 8 + ((lane >> 2) & 3)) * 2 * S + F * 32 + (lane & 3) * 8);
        } else if constexpr (BK == 64) return (uint32_t) ((lane & 15) * 128 + (((lane >> 4) ^ (lane & 7)) * 16));
        else return (uint32_t) ((lane & 15) * 64 + (((lane >> 4) ^ ((lane >> 2) & 3)) * 16));
    }
    template <typename T> static __device__ __forceinline__ v8<T> frag(uint32_t tile, uint32_t fa, int base, int kk) {
        if constexpr (TR) {
            const uint32_t ad = tile + (fa ^ (uint32_t) (base * 2)) + (uint32_t) (kk * 64 * S);
            union { s4 h[2]; v8<T> v; } r;
            r.h[0] = lds_get_tr(ad);
            r.h[1] = lds_get_tr(ad + 8 * S);
            return r.v;
        } else return lds_get<v8<T>>(tile + (fa ^ (uint32_t) (kk * 64)) + (uint32_t) (base * 2 * BK));
    }
};

// One BM x BN tile (output rows x columns) a block of WP x WQ waves, BN / WP columns by BM / WQ rows each; stages of BK
// contraction values, NST of them in LDS.
//
// Eight waves (two a SIMD) work in turns: a barrier ends every part, and the second four waves are one part behind, so that
// on each SIMD one wave multiplies while the other reads its next fragments and starts the DMAs three stages on.
template <typename T, int KIND, bool DUAL, int BM, int BN, int WP, int WQ, int BK, int NST>
__global__ __launch_bounds__(64 * WP * WQ, 2) void k_mm(const MMArgs a) {
    constexpr int NW = WP * WQ, NTH = 64 * NW, FP = BN / WP / 16, FQ = BM / WQ / 16;
    constexpr bool TURNS = NW == 8;
    static_assert(!TURNS || (BK == 32 && NST == 4), "the turns' DMA distance");
    using OP = Operand<KIND != NT, BN, NW, BK>;
    using OQ = Operand<KIND == TN, BM, NW, BK>;
    constexpr int NDMA = OP::N + OQ::N, STAGE = OP::BYTES + OQ::BYTES;
    constexpr int WN = BN / WP;                                  // columns a wave
    constexpr int CH = 512;                                      // TN: contraction rows looked up at a time
    __shared__ __attribute__((aligned(1024))) uint8_t s_mem[NST * STAGE];
    __shared__ int s_pair[KIND == TN ? 1 : BM], s_look[KIND == TN ? 4 * CH : 1];
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
    const int per_part = (K + BK - 1) / BK, nstage = KIND == NN && a.P2 ? 2 * per_part : per_part;
    const char *zero = (const char *) g_zero16;

    // TN by pairs: the operand rows of CH contraction rows at a time, two such chunks in LDS (-1: no row)
    auto look_up = [&](int chunk) {
        if constexpr (KIND == TN) {
            if (!a.order) return;
            for (int i = tid; i < CH; i += NTH) {
                const int k = chunk * CH + i, p = k < K ? pair_of(a, g, k) : -1;
                s_look[(chunk & 1) * CH + i] = p < 0 ? -1 : div_k(p, a.kp, mp);
                s_look[(2 + (chunk & 1)) * CH + i] = p < 0 ? -1 : div_k(p, a.kq, mq);
            }
        }
    };
    auto issue = [&](int s, int buf) {
        const uint32_t tp = lds0 + (uint32_t) buf * STAGE, tq = tp + OP::BYTES;
        if constexpr (KIND == TN) {
#pragma unroll
            for (int i = 0; i < OP::N; ++i) {
                const int k = s * BK + OP::krow(wave, lane, i);
                int r = k < K ? k : -1;
                if (a.order && r >= 0) r = s_look[k & (2 * CH - 1)];
                dma16(r >= 0 ? P.p[i] + r * ldp2 : zero, OP::dst(tp, wave, i));
            }
#pragma unroll
            for (int i = 0; i < OQ::N; ++i) {
                const int k = s * BK + OQ::krow(wave, lane, i);
                int r = k < K ? k : -1;
                if (a.order && r >= 0) r = s_look[2 * CH + (k & (2 * CH - 1))];
                dma16(r >= 0 ? Q.p[i] + r * ldq2 : zero, OQ::dst(tq, wave, i));
            }
        } else {
            int64_t dp = 0, dq = 0;
            int sl = s;
            if (KIND == NN && a.P2 && s >= per_part) {   // the second part's matrices
                sl = s - per_part;
                dp = (const char *) a.P2 - (const char *) a.P;
                dq = (const char *) a.Q2 - (const char *) a.Q;
            }
            dp += (KIND == NT ? 2 * BK : BK * ldp2) * (int64_t) sl;
            dq += 2 * BK * (int64_t) sl;
            const bool full = sl * BK + BK <= K;
#pragma unroll
            for (int i = 0; i < OP::N; ++i) {
                const char *src = P.p[i] + dp;
                if (!full && sl * BK + OP::krow(wave, lane, i) >= K) src = zero;
                dma16(src, OP::dst(tp, wave, i));
            }
#pragma unroll
            for (int i = 0; i < OQ::N; ++i) {
                const char *src = Q.p[i] + dq;
                if (!full && sl * BK + OQ::krow(wave, lane, i) >= K) src = zero;
                dma16(src, OQ::dst(tq, wave, i));
            }
        }
    };

    f4 acc[FP][FQ] = {};
    f4 dbs[KIND == TN ? FQ : 1] = {};
    const bool do_db = KIND == TN && a.db && col == 0 && wp == 0;
    const uint32_t fap = OP::frag_addr(lane), faq = OQ::frag_addr(lane);
    auto read = [&](v8<T> (&fp)[FP], v8<T> (&fq)[FQ], uint32_t tp, int kk) {
#pragma unroll
        for (int j = 0; j < FQ; ++j) fq[j] = OQ::template frag<T>(tp + OP::BYTES, faq, wq * (BM / WQ) + j * 16, kk);
#pragma unroll
        for (int i = 0; i < FP; ++i) fp[i] = OP::template frag<T>(tp, fap, wp * WN + i * 16, kk);
    };
    auto multiply = [&](const v8<T> (&fp)[FP], const v8<T> (&fq)[FQ]) {
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
    };
    if constexpr (KIND == TN) {
        look_up(0);
        look_up(1);
        __syncthreads();
    }
    // one chunk is looked up while the one before is in use: behind its last DMA, before the next chunk's first
    auto look_ahead = [&](int s) {
        if constexpr (KIND == TN) {
            constexpr int SPC = CH / BK;   // stages a chunk
            if (a.order && s % SPC == SPC / 2 && s > SPC) look_up(s / SPC + 1);
        }
    };
    if constexpr (TURNS) {
        // stages behind the last are DMAs of zeros, so that the counts of DMAs in flight stay the same
        for (int s = 0; s < 3; ++s) issue(s, s);
        wait_vm<2 * NDMA>();
        lds_barrier();
        if (wave >= 4) __builtin_amdgcn_s_barrier();
        for (int s = 0; s < nstage; ++s) {
            v8<T> fp[FP], fq[FQ];
            read(fp, fq, lds0 + (uint32_t) (s & 3) * STAGE, 0);
            look_ahead(s);
            issue(s + 3, (s + 3) & 3);
            wait_vm<2 * NDMA>();   // stage s + 1 is in place
            lds_barrier();
            __builtin_amdgcn_sched_barrier(0);
            __builtin_amdgcn_s_setprio(1);
            multiply(fp, fq);
            __builtin_amdgcn_s_setprio(0);
            __builtin_amdgcn_sched_barrier(0);
            lds_barrier();
        }
        if (wave < 4) __builtin_amdgcn_s_barrier();
    } else {
        for (int s = 0; s < NST - 1; ++s)
            if (s < nstage) issue(s, s);
        int buf = 0;
        for (int s = 0; s < nstage; ++s) {
            // this stage has landed for every wave, and every wave is done with the one before
            if (NST > 2 && s + NST - 2 < nstage) wait_vm<(NST - 2) * NDMA>();
            else wait_vm<0>();
            lds_barrier();
            look_ahead(s);
            if (s + NST - 1 < nstage) issue(s + NST - 1, buf == 0 ? NST - 1 : buf - 1);
#pragma unroll
            for (int kk = 0; kk < BK / 32; ++kk) {
                v8<T> fp[FP], fq[FQ];
                read(fp, fq, lds0 + (uint32_t) buf * STAGE, kk);
                multiply(fp, fq);
            }
            buf = buf == NST - 1 ? 0 : buf + 1;
        }
    }
    wait_vm<0>();
    __syncthreads();

    // Epilogue, 16 JP rows of the wave at a time through its own part of the stages (row r's 16-byte piece c at c ^ r), so
    // that a lane holds eight neighbouring columns and a row's lanes write whole lines
    constexpr int PCS = WN / 4, X = PCS < 16 ? PCS - 1 : 15;
    constexpr int LPR = (DUAL ? WN / 2 : WN) / 8, RPI = 64 / LPR;   // lanes a row, rows at a time
    constexpr int FIT = NST * STAGE / (NW * 16 * WN * 4), JP = FIT >= FQ ? FQ : FIT >= 4 && FQ % 4 == 0 ? 4 : FIT >= 2 && FQ % 2 == 0 ? 2 : 1;
    static_assert(FIT >= 1 && FQ % JP == 0, "the epilogue's rows fit the stages");
    const uint32_t own = lds0 + (uint32_t) wave * JP * 16 * WN * 4;
    const int cl = c0 + wp * (CN / WP) + lane % LPR * 8;
#pragma unroll
    for (int j0 = 0; j0 < FQ; j0 += JP) {
#pragma unroll
        for (int j = 0; j < JP; ++j) {
            const uint32_t r = lane & 15;
#pragma unroll
            for (int i = 0; i < FP; ++i)
                *(__attribute__((address_space(3))) f4 *) (uintptr_t) (own + (r + 16 * j) * (WN * 4) + (((uint32_t) (i * 4 + (lane >> 4)) ^ (r & X)) * 16)) = acc[i][j0 + j];
        }
        wave_sync();
#pragma unroll 1
        for (int h = 0; h < 16 * JP; h += RPI) {
            const int r = RPI <= 16 ? h + lane / LPR : h + (lane / LPR) % (16 * JP);
            const int i0 = wq * (BM / WQ) + j0 * 16 + r;
            int row;
            int64_t ob = 0;
            float w = 1.0f;
            if constexpr (KIND == TN) {
                row = r0 + i0 < a.R ? r0 + i0 : -1;
                ob = (int64_t) blockIdx.y * a.ostride;
            } else {
                row = s_pair[i0];
                if (a.wts && row >= 0) w = a.wts[row];
            }
            if (RPI > 16 * JP && lane / LPR >= 16 * JP) row = -1;   // lanes without a row
            auto piece = [&](int c) { return lds_get<f4>(own + (uint32_t) r * (WN * 4) + (((uint32_t) c ^ ((uint32_t) r & X)) * 16)); };
            union { f4 q[2]; float v[8]; } u, g2;
            if constexpr (DUAL) {
                const int c = lane % LPR * 2, at = (c >> 2) * 8 + (c & 3);   // 16 gate columns, 16 up columns, ..
                u.q[0] = piece(at);
                u.q[1] = piece(at + 1);
                g2.q[0] = piece(at + 4);
                g2.q[1] = piece(at + 5);
                if (row >= 0) epi_glu<T, 8>(a, row, cl, u.v, g2.v);
            } else {
                u.q[0] = piece(lane % LPR * 2);
                u.q[1] = piece(lane % LPR * 2 + 1);
                if (row >= 0) epi_store<T, 8>(a, ob, row, cl, u.v, w);
            }
        }
        wave_sync();
    }
    if constexpr (KIND == TN) {
        if (do_db && lane < 16) {
#pragma unroll
            for (int j = 0; j < FQ; ++j) {
                const int row = r0 + wq * (BM / WQ) + j * 16 + lane;
                if (row < a.R) a.db[row] = a.accumulate ? a.db[row] + dbs[j][0] : dbs[j][0];
            }
        }
    }
}

template <typename T, int KIND, bool DUAL, int BM, int BN, int WP, int WQ, int BK, int NST>
static int launch_tile(const MMArgs &a, hipStream_t s, const char *what) {
    const int64_t ncol = (a.N + (DUAL ? BN / 2 : BN) - 1) / (DUAL ? BN / 2 : BN);
    const int64_t items = KIND == TN || !a.egrp ? ((int64_t) a.R + BM - 1) / BM : ((int64_t) a.n_pairs + BM - 1) / BM + a.max_active;
    const int64_t blocks = ncol * items;
    if (blocks <= 0) return HY_OK;
    if (blocks > 0x7fffffffll) { set_error("%s: %lld tiles", what, (long long) blocks); return HY_EBAD_SHAPE; }
    k_mm<T, KIND, DUAL, BM, BN, WP, WQ, BK, NST><<<dim3((uint32_t) blocks, KIND == TN && a.egrp ? (uint32_t) a.n_local : 1u), 64 * WP * WQ, 0, s>>>(a);
    return check_launch(what);
}

} // namespace hy
