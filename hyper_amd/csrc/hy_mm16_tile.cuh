// The tile kernels of the 16-bit matrix products: operands by LDS DMA, 16 x 16 x 32 matrix instructions.
#pragma once
#include "hy_mm16.cuh"

#include <algorithm>
#include <cmath>

namespace hy {

// 16 bytes a lane from per-lane addresses to 1 KB of LDS at `lds` (lane l's bytes at lds + 16 l), in flight when it returns.
// M0 holds the LDS address (named as overwritten, so that the compiler keeps nothing of its own there).
__device__ __forceinline__ void dma16(const char *src, uint32_t lds) {
    asm volatile("s_mov_b32 m0, %1\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %0, off" ::"v"(src), "s"(lds) : "memory", "m0");
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

// How an operand's tile of S rows (or columns) by BK = 64 contraction values lies in LDS, in 16-byte pieces:
//  along the contraction (TR false): row r at r * 128, its piece c at c ^ (r & 7): a fragment read takes one piece of each of 16
//  rows, 16 lanes at a time in different places of 256 bytes
//  across it (TR true): contraction row k at k * 2 S, its pair of pieces u at u ^ F(k), F = k & 3 | bit 3 of k << 2 (S 64:
//  k & 3): a transposing read takes 32 bytes of the rows 8 q + 0..3 (or 4..7) of two quarters q at a time, eight different F
// Both read at 240 bytes a clock and CU (256 is the most).  Rows of 128 bytes are whole lines: 32 values a stage (64 bytes)
// halved the rate at which all CUs together fetch from L2 (67 against 133 bytes / ns and CU).
constexpr int BK = 64;
template <bool TR, int S, int NW> struct Operand {
    static constexpr int N = S * BK / 512 / NW;   // DMAs (of 1 KB) a wave and stage
    static_assert(N * 512 * NW == S * BK, "whole DMAs");
    static constexpr int BYTES = S * BK * 2;
    static constexpr int CPR = TR ? S / 8 : 8, RPI = 64 / CPR;   // pieces a stored row, stored rows a DMA
    const char *p[N];     // the lanes' places in the first stage
    const char *cur[N];   // and in the next one to fetch

    // the DMA's contraction row within the stage (TR) / first contraction value of the lane's piece (not TR)
    static __device__ __forceinline__ int krow(int wave, int lane, int i) {
        if constexpr (TR) return (wave * N + i) * RPI + lane / CPR;
        else return ((lane & 7) ^ (lane >> 3)) * 8;
    }
    // the lane's row (not TR) / first column (TR) within the tile
    static __device__ __forceinline__ int at(int wave, int lane, int i) {
        if constexpr (TR) {
            const int k = krow(wave, lane, i), pc = lane % CPR, F = (k & 3) | (S >= 128 ? (k >> 1) & 4 : 0);
            return (((pc >> 1) ^ F) * 2 + (pc & 1)) * 8;
        } else return (wave * N + i) * RPI + lane / CPR;
    }
    // lane's part of the address of a fragment (16 rows / columns; 32 contraction values)
    static __device__ __forceinline__ uint32_t frag_addr(int lane) {
        if constexpr (TR) {
            const int F = ((lane >> 2) & 3) | (S >= 128 ? (lane >> 2) & 4 : 0);
            return (uint32_t) (((lane >> 4) * 8 + ((lane >> 2) & 3)) * 2 * S + F * 32 + (lane & 3) * 8);
        } else return (uint32_t) ((lane & 15) * 128 + (((lane >> 4) ^ (lane & 7)) * 16));
    }
    // fragment i of the wave's rows / columns from w0 (a multiple of 64, or of 32 with S >= 64), half kk of the stage;
    // fa: frag_addr, `base` the stage's place in LDS
    template <typename T> static __device__ __forceinline__ v8<T> frag(uint32_t base, uint32_t fa, int w0, int i, int kk) {
        if constexpr (TR) {
            const uint32_t ad = base + (fa ^ (uint32_t) ((w0 + i * 16) * 2));
            union { s4 h[2]; v8<T> v; } r;
            r.h[0] = lds_get_tr(ad + (uint32_t) (kk * 64 * S));
            r.h[1] = lds_get_tr(ad + (uint32_t) (kk * 64 * S + 8 * S));
            return r.v;
        } else return lds_get<v8<T>>(base + (fa ^ (uint32_t) (kk * 64)) + (uint32_t) (w0 * 128) + (uint32_t) (i * 2048));
    }
};
__device__ __forceinline__ void mfma_acc(f4 &c, v8<bf16> a, v8<bf16> b) { asm("v_mfma_f32_16x16x32_bf16 %0, %1, %2, %0" : "+a"(c) : "v"(a), "v"(b)); }
__device__ __forceinline__ void mfma_acc(f4 &c, v8<f16> a, v8<f16> b) { asm("v_mfma_f32_16x16x32_f16 %0, %1, %2, %0" : "+a"(c) : "v"(a), "v"(b)); }

// One BM x BN tile (output rows x columns, from r0 and column tile col on) by a block of WP x WQ waves, BN / WP columns by
// BM / WQ rows each; stages of 64 contraction values, NST of them in LDS, one barrier a stage.
//
// A stage is two halves of 32 values.  While one half's products run, the wave reads the next half's fragments into the other
// registers and, behind the barrier, starts the DMAs of the stage NST on (whose place every wave has read by then): the reads
// and DMAs go between the products one at a time, since a wave issues in order and two or three instructions hide behind a
// product of 16 clocks.
template <int KIND, int BM, int BN, int WP, int WQ, int NST> struct TileLds {   // bytes of the stages
    static constexpr int STAGES = NST * (Operand<KIND != NT, BN, WP * WQ>::BYTES + Operand<KIND == TN, BM, WP * WQ>::BYTES);
};
constexpr int LOOK = 512;   // TN: contraction rows looked up at a time
template <typename T, int KIND, bool DUAL, int BM, int BN, int WP, int WQ, int NST>
__device__ __forceinline__ void mm_tile(const MMArgs &a, const Group &g, int r0, int col, uint8_t *s_mem, int *s_pair, int *s_look) {
    constexpr int NW = WP * WQ, NTH = 64 * NW, FP = BN / WP / 16, FQ = BM / WQ / 16;
    constexpr bool WIDE = FP * FQ == 64;   // 256 sums a lane: in the accumulation registers
    using OP = Operand<KIND != NT, BN, NW>;
    using OQ = Operand<KIND == TN, BM, NW>;
    constexpr int NDMA = OP::N + OQ::N, STAGE = OP::BYTES + OQ::BYTES;
    constexpr int WN = BN / WP;                                  // columns a wave
    constexpr int CH = LOOK;
    const int tid = threadIdx.x, wave = __builtin_amdgcn_readfirstlane(tid >> 6), lane = tid & 63, wp = wave % WP, wq = wave / WP;
    constexpr int CN = DUAL ? BN / 2 : BN;   // output columns a tile
    const int c0 = col * CN;
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
            P.p[i] = Pb + c * 2 + (KIND == TN && a.order ? 0 : (OP::krow(wave, lane, i) + (KIND == TN ? g.start : 0)) * ldp2);
        }
    }
#pragma unroll
    for (int i = 0; i < OQ::N; ++i) {
        const int at = OQ::at(wave, lane, i);
        if constexpr (KIND == TN) {
            const int r = r0 + at < a.R ? r0 + at : r0;
            Q.p[i] = (const char *) a.Q + r * 2 + (a.order ? 0 : (OQ::krow(wave, lane, i) + g.start) * ldq2);
        } else {
            const int p = max(s_pair[at], 0);
            Q.p[i] = (const char *) a.Q + div_k(p, a.kq) * ldq2 + OQ::krow(wave, lane, i) * 2;
        }
    }
    const uint32_t lds0 = (uint32_t) __builtin_amdgcn_readfirstlane((int) lds_addr(s_mem));
    const int per_part = (K + BK - 1) / BK, nstage = KIND == NN && a.P2 ? 2 * per_part : per_part;
    const char *zero = (const char *) g_zero16;

    // TN by pairs: the operand rows of CH contraction rows at a time, two such chunks in LDS (-1: no row)
    auto look_up = [&](int chunk) {
        if constexpr (KIND == TN) {
            if (!a.order) return;
            for (int i = tid; i < CH; i += NTH) {
                const int k = chunk * CH + i, p = k < K ? pair_of_expert(a, g, k) : -1;
                s_look[(chunk & 1) * CH + i] = p < 0 ? -1 : div_k(p, a.kp);
                s_look[(2 + (chunk & 1)) * CH + i] = p < 0 ? -1 : div_k(p, a.kq);
            }
        }
    };
    // The places to fetch stage s from.  They move on by a constant distance, but where a part begins or ends: at stage
    // `event` they are made anew.  By pairs (TN) every stage makes them anew.
    int64_t step_p = 0, step_q = 0;
    int event = 0;
    auto places = [&](int s) {
        if (KIND == TN && a.order) {
            if constexpr (KIND == TN) {
#pragma unroll
                for (int i = 0; i < OP::N; ++i) {
                    const int r = s_look[(s * BK + OP::krow(wave, lane, i)) & (2 * CH - 1)];
                    P.cur[i] = s < nstage && r >= 0 ? P.p[i] + r * ldp2 : zero;
                }
#pragma unroll
                for (int i = 0; i < OQ::N; ++i) {
                    const int r = s_look[2 * CH + ((s * BK + OQ::krow(wave, lane, i)) & (2 * CH - 1))];
                    Q.cur[i] = s < nstage && r >= 0 ? Q.p[i] + r * ldq2 : zero;
                }
            }
            return;
        }
        if (s < event) return;
        int64_t dp = 0, dq = 0;
        int sl = s;
        if (KIND == NN && a.P2 && s >= per_part) {   // the second part's matrices
            sl = s - per_part;
            dp = (const char *) a.P2 - (const char *) a.P;
            dq = (const char *) a.Q2 - (const char *) a.Q;
        }
        const int left = s < nstage ? K - sl * BK : 0;   // contraction values left of the part
        step_p = left > 0 ? (KIND == NT ? 2 * BK : BK * ldp2) : 0;
        step_q = left > 0 ? (KIND == TN ? BK * ldq2 : 2 * BK) : 0;
        dp += (KIND == NT ? 2 * BK : BK * ldp2) * (int64_t) sl;
        dq += (KIND == TN ? BK * ldq2 : 2 * BK) * (int64_t) sl;
#pragma unroll
        for (int i = 0; i < OP::N; ++i) P.cur[i] = OP::krow(wave, lane, i) < left ? P.p[i] + dp : zero;
#pragma unroll
        for (int i = 0; i < OQ::N; ++i) Q.cur[i] = OQ::krow(wave, lane, i) < left ? Q.p[i] + dq : zero;
        // whole stages follow up to the part's last, partial one (or the next part)
        event = left <= 0 ? 0x7fffffff : left < 2 * BK ? s + 1 : s + left / BK;
    };
    auto fetch = [&](int i, uint32_t stage) {   // the i-th DMA of the stage at LDS address `stage`
        if (i < OP::N) {
            dma16(P.cur[i < OP::N ? i : 0], stage + (uint32_t) (wave * OP::N + i) * 1024);
            P.cur[i < OP::N ? i : 0] += step_p;
        } else {
            const int j = i < OP::N ? 0 : i - OP::N;
            dma16(Q.cur[j], stage + OP::BYTES + (uint32_t) (wave * OQ::N + j) * 1024);
            Q.cur[j] += step_q;
        }
    };

    f4 acc[FP][FQ] = {};
    f4 dbs[KIND == TN ? FQ : 1] = {};
    const bool do_db = KIND == TN && a.db && col == 0 && wp == 0;
    const uint32_t fap = OP::frag_addr(lane), faq = OQ::frag_addr(lane);
    v8<T> fp[2][FP], fq[2][FQ];
    // the o-th fragment of half kk: the first column's, the rows', then the other columns' (the order of their use)
    auto read = [&](int o, int kk, uint32_t bp, uint32_t bq) {
        if (o == 0) fp[kk][0] = OP::template frag<T>(bp, fap, wp * WN, 0, kk);
        else if (o <= FQ) fq[kk][o <= FQ && o > 0 ? o - 1 : 0] = OQ::template frag<T>(bq, faq, wq * (BM / WQ), o - 1, kk);
        else fp[kk][o > FQ ? o - FQ : 0] = OP::template frag<T>(bp, fap, wp * WN, o - FQ, kk);
    };
    auto product = [&](int m, int kk) {
        if constexpr (WIDE) mfma_acc(acc[m / FQ][m % FQ], fp[kk][m / FQ], fq[kk][m % FQ]);
        else acc[m / FQ][m % FQ] = mfma16(fp[kk][m / FQ], fq[kk][m % FQ], acc[m / FQ][m % FQ]);
    };
    auto db_product = [&](int kk) {   // the rows' sums as a product with ones
        if constexpr (KIND == TN) {
            if (do_db) {
                v8<T> one;
#pragma unroll
                for (int e = 0; e < 8; ++e) one[e] = (T) 1.0f;
#pragma unroll
                for (int j = 0; j < FQ; ++j) dbs[j] = mfma16(one, fq[kk][j], dbs[j]);
            }
        }
    };
    constexpr int NM = FP * FQ, NR = FP + FQ;
    if constexpr (KIND == TN) {
        look_up(0);
        look_up(1);
        __syncthreads();
    }
    // stages behind the last are DMAs of zeros, so that the counts of DMAs in flight stay the same
    for (int s = 0; s < NST; ++s) {
        places(s);
#pragma unroll
        for (int i = 0; i < NDMA; ++i) fetch(i, lds0 + (uint32_t) s * STAGE);
    }
    wait_vm<(NST - 1) * NDMA>();
    lds_barrier();
#pragma unroll
    for (int o = 0; o < NR; ++o) read(o, 0, lds0, lds0 + OP::BYTES);
    uint32_t at = lds0;
    for (int s = 0; s < nstage; ++s) {
        uint32_t nx = at + STAGE;
        if (nx == lds0 + NST * STAGE) nx = lds0;
        if constexpr (KIND == TN) {
            // one chunk is looked up while the one before is in use: behind its last DMA, before the next chunk's first
            constexpr int SPC = CH / BK;   // stages a chunk
            static_assert(KIND != TN || NST < SPC / 2, "a chunk is in place before its first DMA");
            if (a.order && s % SPC == SPC / 2 && s > SPC) look_up(s / SPC + 1);
        }
        places(s + NST);
        __builtin_amdgcn_sched_barrier(0);
        uint32_t bp = at, bq = at + OP::BYTES;
#pragma unroll
        for (int m = 0; m < NM; ++m) {
            product(m, 0);
#pragma unroll
            for (int o = min(NR, m * NR * 3 / (NM * 2)); o < min(NR, (m + 1) * NR * 3 / (NM * 2)); ++o) read(o, 1, bp, bq);   // done by two thirds: the barrier waits for them
            __builtin_amdgcn_sched_barrier(0);
        }
        db_product(0);
        wait_vm<(NST - 2) * NDMA>();   // stage s + 1 is in place
        lds_barrier();                 // for every wave, and every wave has read this one
        bp = nx;
        bq = nx + OP::BYTES;
        constexpr int NO = NR + NDMA;
#pragma unroll
        for (int m = 0; m < NM; ++m) {
            product(m, 1);
#pragma unroll
            for (int o = m * NO / NM; o < (m + 1) * NO / NM; ++o) {
                // reads and DMAs in turn
                const int rd = (o + 1) * NR / NO, rd0 = o * NR / NO;
                if (rd > rd0) read(rd0, 0, bp, bq);
                else fetch(o - rd0, at);
            }
            __builtin_amdgcn_sched_barrier(0);
        }
        db_product(1);
        at = nx;
    }
    if constexpr (WIDE) {   // the last products end before their sums are read
        asm volatile("s_nop 15\n\ts_nop 15" ::: "memory");
#pragma unroll
        for (int i = 0; i < FP; ++i)
#pragma unroll
            for (int j = 0; j < FQ; ++j) asm volatile("" : "+a"(acc[i][j]));
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
    const int64_t ob = KIND == TN ? (int64_t) g.le * a.ostride : 0;
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
        auto row_of = [&](int r) -> int {   // the output row of the wave's row r of this pass (-1: none)
            const int i0 = wq * (BM / WQ) + j0 * 16 + r;
            if constexpr (KIND == TN) return r0 + i0 < a.R ? r0 + i0 : -1;
            else return s_pair[i0];
        };
        auto piece = [&](int r, int c) { return lds_get<f4>(own + (uint32_t) r * (WN * 4) + (((uint32_t) c ^ ((uint32_t) r & X)) * 16)); };
        const int pc = DUAL ? (lane % LPR >> 1) * 8 + (lane % LPR * 2 & 3) : lane % LPR * 2;   // the lane's first piece (gated: 16 gate, 16 up, ..)
        if (a.vec && cl + 8 <= a.N) {
            // U rows at a time, so that their reads and stores are in flight together
            constexpr int NIT = 16 * JP / RPI > 0 ? 16 * JP / RPI : 1, U = NIT % 4 == 0 ? 4 : NIT % 2 == 0 ? 2 : 1;
#pragma unroll 1
            for (int h = 0; h < NIT * RPI; h += U * RPI) {
                float v[U][8];
                int row[U];
#pragma unroll
                for (int u = 0; u < U; ++u) {
                    const int r = (h + u * RPI + lane / LPR) % (16 * JP);
                    row[u] = RPI > 16 * JP && lane / LPR >= 16 * JP ? -1 : row_of(r);
                    const f4 p0 = piece(r, pc), p1 = piece(r, pc + 1);
#pragma unroll
                    for (int e = 0; e < 4; ++e) { v[u][e] = p0[e]; v[u][e + 4] = p1[e]; }
                }
                if constexpr (DUAL) {
                    float w[U][8];
#pragma unroll
                    for (int u = 0; u < U; ++u) {
                        const int r = (h + u * RPI + lane / LPR) % (16 * JP);
                        const f4 p0 = piece(r, pc + 4), p1 = piece(r, pc + 5);
#pragma unroll
                        for (int e = 0; e < 4; ++e) { w[u][e] = p0[e]; w[u][e + 4] = p1[e]; }
                    }
                    if (a.g) {
#pragma unroll
                        for (int u = 0; u < U; ++u)
                            if (row[u] >= 0) {
                                put_n<T, 8>(a.g, row[u] * a.ldo + cl, v[u], 8, false, true);
                                put_n<T, 8>(a.u, row[u] * a.ldo + cl, w[u], 8, false, true);
                            }
                    }
                    mm_limit<U * 8>(&v[0][0], &w[0][0], a.clamp);
#pragma unroll
                    for (int u = 0; u < U; ++u)
#pragma unroll
                        for (int e = 0; e < 8; ++e) v[u][e] = mm_swiglu(v[u][e], w[u][e]);
                } else {
                    if (a.bias) {
                        const f4 *b = (const f4 *) (a.bias + cl);
                        float bb[8];
                        if (a.bias16) {
                            const f4 b0 = b[0], b1 = b[1];
#pragma unroll
                            for (int e = 0; e < 4; ++e) { bb[e] = b0[e]; bb[e + 4] = b1[e]; }
                        } else {
#pragma unroll
                            for (int e = 0; e < 8; ++e) bb[e] = a.bias[cl + e];
                        }
#pragma unroll
                        for (int u = 0; u < U; ++u)
#pragma unroll
                            for (int e = 0; e < 8; ++e) v[u][e] += bb[e];
                    }
                    if (a.z) {
#pragma unroll
                        for (int u = 0; u < U; ++u) if (row[u] >= 0) put_n<T, 8>(a.z, row[u] * a.ldz + cl, v[u], 8, false, true);
                    }
                    switch (a.act) {
                    case HY_ACT_RELU: act_n<HY_ACT_RELU, U * 8>(&v[0][0]); break;
                    case HY_ACT_SILU: act_n<HY_ACT_SILU, U * 8>(&v[0][0]); break;
                    case HY_ACT_GELU: act_n<HY_ACT_GELU, U * 8>(&v[0][0]); break;
                    case HY_ACT_GELU_TANH: act_n<HY_ACT_GELU_TANH, U * 8>(&v[0][0]); break;
                    }
                    if (a.wts) {
#pragma unroll
                        for (int u = 0; u < U; ++u) {
                            const float w = row[u] >= 0 ? a.wts[row[u]] : 0.0f;
#pragma unroll
                            for (int e = 0; e < 8; ++e) v[u][e] *= w;
                        }
                    }
                    if (a.resid) {
#pragma unroll
                        for (int u = 0; u < U; ++u) if (row[u] >= 0) add_n<T, 8>(a.resid, row[u] * a.ldr + cl, v[u], 8, a.out_f32, true);
                    }
                    if (a.accumulate) {
#pragma unroll
                        for (int u = 0; u < U; ++u) if (row[u] >= 0) add_n<T, 8>(a.out, ob + row[u] * a.ldo + cl, v[u], 8, a.out_f32, true);
                    }
                }
#pragma unroll
                for (int u = 0; u < U; ++u) if (row[u] >= 0) put_n<T, 8>(a.out, ob + row[u] * a.ldo + cl, v[u], 8, a.out_f32, true);
            }
        } else if (cl < a.N) {   // the last columns, or matrices that cannot be moved in 16-byte pieces
#pragma unroll 1
            for (int h = 0; h < 16 * JP; h += RPI) {
                const int r = (h + lane / LPR) % (16 * JP), row = RPI > 16 * JP && lane / LPR >= 16 * JP ? -1 : row_of(r);
                if (row < 0) continue;
                union { f4 q[2]; float v[8]; } u, g2;
                u.q[0] = piece(r, pc);
                u.q[1] = piece(r, pc + 1);
                if constexpr (DUAL) {
                    g2.q[0] = piece(r, pc + 4);
                    g2.q[1] = piece(r, pc + 5);
                    epi_glu<T, 8>(a, row, cl, u.v, g2.v);
                } else epi_store<T, 8>(a, ob, row, cl, u.v, a.wts ? a.wts[row] : 1.0f);
            }
        }
        wave_sync();
    }
    if constexpr (KIND == TN) {
        if (do_db && lane < 16) {
#pragma unroll
            for (int j = 0; j < FQ; ++j) {
                const int row = r0 + wq * (BM / WQ) + j * 16 + lane;
                if (row < a.R) {
                    float *d = a.db + (a.parts > 1 ? (int64_t) g.le * a.R : 0) + row;
                    *d = a.accumulate ? *d + dbs[j][0] : dbs[j][0];
                }
            }
        }
    }
}

// A block's tile.  Groups (and matrices) end inside a tile: where half or a quarter of its rows are left, a smaller tile of the same
// columns takes them; so it does where the tiles left for the CUs' last turn are shared out (8192 x 4608 outputs of 4096 values, 576 tiles on 256
// CUs: 264 -> 236 us; 4100 x 4096: 155 -> 141).
template <typename T, int KIND, bool DUAL, int BM, int BN, int WP, int WQ, int NST>
__global__ __launch_bounds__(64 * WP * WQ, BM * BN / (WP * WQ) > 8192 ? 1 : 2) void k_mm(const MMArgs a) {
    constexpr int NTH = 64 * WP * WQ, CN = DUAL ? BN / 2 : BN;
    __shared__ __attribute__((aligned(1024))) uint8_t s_mem[TileLds<KIND, BM, BN, WP, WQ, NST>::STAGES];
    __shared__ int s_pair[KIND == TN ? 1 : BM], s_look[KIND == TN ? 4 * LOOK : 1];
    const int ncol = (a.N + CN - 1) / CN;
    Group g;
    int tile, col = 0, part = -1;
    if constexpr (KIND == TN) {
        const int rows = (a.R + BM - 1) / BM, t = xcd_tile(blockIdx.x, (uint32_t) rows * (uint32_t) ncol);
        if (t < 0) return;
        band_tile<4>(t, rows, ncol, tile, col);
        if (a.parts > 1) {
            const int start = (int) blockIdx.y * a.part_len;
            g = Group{(int) blockIdx.y, start, min(a.part_len, a.K - start)};
        } else g = find_expert<NTH>(a, blockIdx.y);
    } else if (!find_tile<NTH, BM>(a, ncol, BM == 64 && a.spread, g, tile, col, part)) return;
    int r0 = tile * BM, left = g.cnt - r0;
    if constexpr (KIND != TN && BM >= 128) {
        if (part >= 0) {   // this block's rows of the tile
            r0 += part * (BM / a.split);
            left = min(left - part * (BM / a.split), BM / a.split);
            if (left <= 0) return;
        }
        if (left <= BM / 4) return mm_tile<T, KIND, DUAL, BM / 4, BN, BM == 256 ? 4 : 2, BM == 256 ? 1 : 2, 3>(a, g, r0, col, s_mem, s_pair, s_look);
        if (left <= BM / 2) return mm_tile<T, KIND, DUAL, BM / 2, BN, 2, 2, 2>(a, g, r0, col, s_mem, s_pair, s_look);
    }
    mm_tile<T, KIND, DUAL, BM, BN, WP, WQ, NST>(a, g, r0, col, s_mem, s_pair, s_look);
}

template <typename T, int KIND, bool DUAL, int BM, int BN, int WP, int WQ, int NST>
static int launch_tile(MMArgs a, hipStream_t s, const char *what) {
    const int64_t ncol = (a.N + (DUAL ? BN / 2 : BN) - 1) / (DUAL ? BN / 2 : BN);
    const int64_t items = KIND == TN || !a.egrp ? ((int64_t) a.R + BM - 1) / BM : ((int64_t) a.n_pairs + BM - 1) / BM + a.max_active;
    a.spread = KIND != TN && BM == 64 && a.egrp;   // (fewer rows: every group is one row tile, and in order is 4 to 8 % faster)
    a.split = KIND != TN && BM == 256 && !a.egrp ? split_parts(ncol * items) : 1;
    const int64_t per = (ncol * items + 7) / 8;   // tiles of an XCD
    const int64_t blocks = a.split > 1 ? 8 * ((per & ~31ll) + (per & 31) * a.split) : a.spread ? (ncol + 7) / 8 * 8 * items : ncol * items;   // an XCD has at most ncol / 8, rounded up, of a group's columns
    if (blocks <= 0) return HY_OK;
    if (const int rc = check_blocks(what, blocks)) return rc;
    k_mm<T, KIND, DUAL, BM, BN, WP, WQ, NST><<<dim3((uint32_t) blocks, KIND == TN ? (uint32_t) (a.parts > 1 ? a.parts : std::max(1, a.n_local)) : 1u), 64 * WP * WQ, 0, s>>>(a);
    return check_launch(what);
}

// ------------------------------------------------------------------ which tile

// A tile's rows, columns, tiles that run at once (256 CUs times those that fit a CU), and its cost in microseconds: of one stage
// when few tiles run, when 256 run, when all of `slots` run, and of its start and epilogue.  Measured on bf16 forward products:
// 4096^3 (as many turns of full slots as tiles ask), 256 tiles and fewer of 2048 .. 4096 contraction values.
struct TileCost { int bm, bn, slots; float few, t256, full, ends; };
constexpr TileCost T256x256{256, 256, 256, 1.37f, 2.07f, 2.07f, 11.0f}, T128x128{128, 128, 512, 0.66f, 0.88f, 1.19f, 5.0f},
    T64x128{64, 128, 512, 0.345f, 0.40f, 0.708f, 3.2f}, T64x64{64, 64, 512, 0.26f, 0.272f, 0.5f, 2.5f},
    T32x128{32, 128, 512, 0.286f, 0.30f, 0.574f, 2.2f}, T32x64{32, 64, 512, 0.20f, 0.22f, 0.334f, 2.0f};

// turns of full slots, then what is left.  Grouped rows are a guess: the pairs spread evenly over the groups, a tile begun in
// each (half a tile over; a fifth where smaller tiles take the group's end, and then no group costs less than 0.4 of a tile).
inline float tile_cost(const TileCost &t, const MMArgs &a, int kind, bool dual, int parts = 1) {
    const int cn = dual ? t.bn / 2 : t.bn;
    const double ncol = (a.N + cn - 1) / cn, groups = a.egrp ? std::max(1, std::min({a.max_active, a.n_expert, a.n_pairs})) : 1;
    double rows = kind == TN ? (double) ((a.R + t.bm - 1) / t.bm) * (a.egrp ? a.n_local : 1)
                  : !a.egrp  ? (double) (((int64_t) a.R + t.bm - 1) / t.bm)
                             : groups * (t.bm >= 128 ? std::max(0.4, a.n_pairs / groups / t.bm + 0.22) : std::max(1.0, a.n_pairs / groups / t.bm + 0.5));
    const double stages = kind == TN ? (a.egrp ? a.n_pairs / groups : a.K) / BK + 1 : (double) (a.K + BK - 1) / BK * (kind == NN && a.P2 ? 2 : 1);
    if (kind != TN && a.egrp && t.bm >= 128 && a.n_pairs <= 40 * groups) return 1e30f;   // the weights' bytes bound these: 64 rows
    const double tiles = rows * ncol * parts, whole = std::floor(tiles / t.slots), left = tiles - whole * t.slots;
    double part = 0;
    if (left >= 1) {
        const double st = left <= 256 ? t.few + (t.t256 - t.few) * left / 256 : t.t256 + (t.full - t.t256) * (left - 256) / std::max(1, t.slots - 256);
        part = stages * st + t.ends;
        if (kind != TN && t.bm == 256 && !a.egrp) part *= left <= 64 ? 0.4f : left <= 128 ? 0.66f : 1.0f;   // shared out
    }
    return (float) (whole * (stages * t.full + t.ends) + part);
}
// the cheapest of the tiles
template <int N> inline int cheapest(const TileCost (&t)[N], const MMArgs &a, int kind, bool dual) {
    int best = 0;
    float least = tile_cost(t[0], a, kind, dual);
    for (int i = 1; i < N; ++i) {
        const float c = tile_cost(t[i], a, kind, dual);
        if (c < least) { least = c; best = i; }
    }
    return best;
}

} // namespace hy
