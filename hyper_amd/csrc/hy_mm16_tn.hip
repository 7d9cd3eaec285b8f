// Gradients of the weights: dz^T x, plain and grouped by expert.
#include "hy_mm16_tile.cuh"

namespace hy {

// 64 x 128: 4096 rows of 2048 x 2048 (512 tiles) 66 us, 8192 rows of 2048 x 1024 (256 tiles) 62 us
constexpr TileCost TILES[] = {T256x256, T128x128, {64, 128, 512, 0.36f, 0.46f, 0.97f, 3.2f}};

// Experts' gradients of few rows each (256 pairs: four stages a 256 x 256 tile): alone, a tile's start (group, pairs, first rows)
// and end take longer than its products.  Here a block goes through up to `nct` column tiles of one expert and row tile: the
// group and the pairs' rows are looked up once, the stages of the tiles follow one another without a break, and a tile's sums go
// out from the registers while the next tile's first stages are on their way.
constexpr int PAIRS = 1024;   // pairs of an expert that a block keeps in LDS; an expert with more has a block a tile

// a sum moved to an ordinary register here and not before (moved ahead of their use, they run out of registers)
__device__ __forceinline__ float acc_read(float s) {
    float v;
    asm volatile("v_accvgpr_read_b32 %0, %1" : "=v"(v) : "a"(s));
    return v;
}
// The sums of a wave's 128 columns and 16 FQ rows.  A lane has four neighbouring columns of each fragment.  16 bits: it trades four
// of one fragment for four of the next, and stores eight.  fp32: rows r + 8 of one fragment are traded for rows r of the next, so
// that eight lanes write 128 bytes of a row.
template <typename T, bool F32, int FP, int FQ>
__device__ __forceinline__ void store_sums(const MMArgs &a, f4 (&acc)[FP][FQ], int64_t ob, int row0, int c0, int lane) {
    typedef uint32_t u4 __attribute__((ext_vector_type(4)));
    const uint32_t ldo = (uint32_t) a.ldo;
#pragma unroll
    for (int j = 0; j < FQ; ++j) {
        asm volatile("" : "+v"(lane));   // (the places are made here: no registers to keep them)
        const int rj = row0 + j * 16;
        if constexpr (F32) {
            const bool lo = (lane & 8) == 0;
            const int r = lane & 7, c4 = (lo ? 0 : 16) + (lane >> 4) * 4;
            float *o = (float *) a.out + (ob + (int64_t) rj * a.ldo + c0);
            const uint32_t at = (uint32_t) r * ldo + (uint32_t) c4;   // (below 2^25)
            const bool in0 = rj + r < a.R, in1 = rj + r + 8 < a.R;
#pragma unroll
            for (int i = 0; i < FP; i += 2) {
                f4 x, y;
#pragma unroll
                for (int e = 0; e < 4; ++e) { x[e] = acc_read(acc[i][j][e]); y[e] = acc_read(acc[i + 1][j][e]); }
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const float t = __builtin_bit_cast(float, __builtin_amdgcn_mov_dpp(__builtin_bit_cast(int, lo ? y[e] : x[e]), 0x128, 0xf, 0xf, true));   // eight lanes on within 16
                    x[e] = lo ? x[e] : t;
                    y[e] = lo ? t : y[e];
                }
                if (c0 + c4 + i * 16 < a.N) {
                    f4 *p = (f4 *) (o + (at + i * 16)), *q = (f4 *) (o + (at + 8 * ldo + i * 16));
                    if (a.accumulate) {
                        if (in0) x += *p;
                        if (in1) y += *q;
                    }
                    if (in0) *p = x;
                    if (in1) *q = y;
                }
                __builtin_amdgcn_sched_barrier(0);
            }
        } else {
            const int r = lane & 15, c8 = ((lane >> 4) & 1) * 16 + (lane >> 5) * 8;
            T *o = (T *) a.out + (ob + (int64_t) rj * a.ldo + c0);
            const uint32_t at = (uint32_t) r * ldo + (uint32_t) c8;
            const bool in = rj + r < a.R;
#pragma unroll
            for (int i = 0; i < FP; i += 2) {
                union { T t[4]; uint32_t w[2]; } x, y;
#pragma unroll
                for (int e = 0; e < 4; ++e) { x.t[e] = (T) acc[i][j][e]; y.t[e] = (T) acc[i + 1][j][e]; }
                const auto s0 = __builtin_amdgcn_permlane16_swap(x.w[0], y.w[0], false, false);   // x's odd sixteens for y's even ones
                const auto s1 = __builtin_amdgcn_permlane16_swap(x.w[1], y.w[1], false, false);
                if (in && c0 + c8 + i * 16 < a.N) *(u4 *) (o + (at + i * 16)) = u4{s0[0], s1[0], s0[1], s1[1]};
            }
        }
        __builtin_amdgcn_sched_barrier(0);
    }
}

template <typename T, bool F32> __global__ __launch_bounds__(256, 1) void k_gradients(const MMArgs a, const int nct) {
    constexpr int FP = 8, FQ = 8, NM = FP * FQ, NR = FP + FQ, NST = 2, CN = 256;
    using O = Operand<true, 256, 4>;   // both operands
    constexpr int NDMA = 2 * O::N, STAGE = 2 * O::BYTES;
    __shared__ __attribute__((aligned(1024))) uint8_t s_mem[NST * STAGE];
    __shared__ int s_look[2 * PAIRS];
    const int ncol = (a.N + CN - 1) / CN, rows = (a.R + 255) / 256, chunks = (ncol + nct - 1) / nct;
    // the chunks' first tiles come first, all of an expert on one XCD; then the tiles between, which only long groups have
    int le, tile, col;
    const uint32_t per = (uint32_t) (rows * chunks), firsts = per * (uint32_t) a.n_local;
    const bool first = blockIdx.x < firsts;
    if (first) {
        const uint32_t whole = (uint32_t) a.n_local & ~7u;
        uint32_t t;
        if (blockIdx.x < whole * per) {
            le = (int) ((blockIdx.x & 7) + (blockIdx.x >> 3) / per * 8);
            t = (blockIdx.x >> 3) % per;
        } else {
            const uint32_t r = blockIdx.x - whole * per;
            le = (int) (whole + r / per);
            t = r % per;
        }
        tile = (int) t % rows;
        col = (int) t / rows * nct;
    } else {
        const uint32_t rest = (uint32_t) (rows * (ncol - chunks)), r = blockIdx.x - firsts;
        le = (int) (r / rest);
        const uint32_t t = r % rest;
        tile = (int) (t % (uint32_t) rows);
        const int c = (int) (t / (uint32_t) rows);   // the c-th of the columns that are no multiple of nct
        col = c / (nct - 1) * nct + c % (nct - 1) + 1;
    }
    const Group g = find_expert<256>(a, le);
    const int K = g.cnt, r0 = tile * 256;
    if (K > PAIRS) return mm_tile<T, TN, false, 256, 256, 2, 2, NST>(a, g, r0, col, s_mem, nullptr, s_look);
    if (!first) return;
    const int nt = min(nct, ncol - col), nstage = max((K + BK - 1) / BK, 1);   // (no pairs: a stage of zeros)

    const int tid = threadIdx.x, wave = __builtin_amdgcn_readfirstlane(tid >> 6), lane = tid & 63, wp = wave & 1, wq = wave >> 1;
    for (int i = tid; i < nstage * BK; i += 256) {   // the pairs' rows; -1: none
        const int p = i < K ? pair_of_expert(a, g, i) : -1;
        s_look[i] = p < 0 ? -1 : div_k(p, a.kp);
        s_look[PAIRS + i] = p < 0 ? -1 : div_k(p, a.kq);
    }
    const uint32_t lds0 = (uint32_t) __builtin_amdgcn_readfirstlane((int) lds_addr(s_mem));
    const uint32_t pitch_p = (uint32_t) a.ldp * 2, pitch_q = (uint32_t) a.ldq * 2;
    const char *zero = (const char *) g_zero16;
    int ft = 0, fs = 0;   // the next stage to fetch: stage fs of column tile ft (nt: none)
    // row and columns of the i-th DMA's lanes; columns outside the matrices are the tile's first (never stored)
    int seen[NDMA];
    auto look = [&](int i) {
        const int k = fs * BK + O::krow(wave, lane, i % O::N);
        seen[i] = ft < nt ? s_look[i < O::N ? k : PAIRS + k] : -1;
    };
    auto fetch = [&](int i, uint32_t stage) {
        int ln = lane;
        asm volatile("" : "+v"(ln));   // (made at their use: no registers to keep them)
        const int at = O::at(wave, ln, i % O::N), c = (i < O::N ? (col + ft) * CN : r0) + at;
        const int cc = c < (i < O::N ? a.N : a.R) ? c : c - at;
        const char *base = (const char *) (i < O::N ? a.P : a.Q);
        const char *src = base + ((uint64_t) (uint32_t) seen[i] * (i < O::N ? pitch_p : pitch_q) + (uint32_t) cc * 2);   // (pitches below 2^31)
        dma16(seen[i] >= 0 ? src : zero, stage + (i < O::N ? 0 : O::BYTES) + (uint32_t) (wave * O::N + i % O::N) * 1024);
    };
    auto fetched = [&]() {
        if (++fs == nstage) { fs = 0; ft = min(ft + 1, nt); }
    };

    f4 acc[FP][FQ] = {};
    const uint32_t fap0 = O::frag_addr(lane), faq0 = fap0;
    v8<T> fp[2][FP], fq[2][FQ];
    auto read = [&](int o, int kk, uint32_t at) {   // as in mm_tile
        uint32_t fa = o > 0 && o <= FQ ? faq0 : fap0;
        asm volatile("" : "+v"(fa));
        if (o == 0) fp[kk][0] = O::template frag<T>(at, fa, wp * 128, 0, kk);
        else if (o <= FQ) fq[kk][o <= FQ && o > 0 ? o - 1 : 0] = O::template frag<T>(at + O::BYTES, fa, wq * 128, o - 1, kk);
        else fp[kk][o > FQ ? o - FQ : 0] = O::template frag<T>(at, fa, wp * 128, o - FQ, kk);
    };
    __syncthreads();
    for (int s = 0; s < NST; ++s) {
#pragma unroll
        for (int i = 0; i < NDMA; ++i) look(i);
#pragma unroll
        for (int i = 0; i < NDMA; ++i) fetch(i, lds0 + (uint32_t) s * STAGE);
        fetched();
    }
    wait_vm<(NST - 1) * NDMA>();
    lds_barrier();
#pragma unroll
    for (int o = 0; o < NR; ++o) read(o, 0, lds0);
    uint32_t at = lds0;
    const int64_t ob = (int64_t) g.le * a.ostride;
    for (int t = 0; t < nt; ++t) {
        for (int s = 0; s < nstage; ++s) {
            const uint32_t nx = at == lds0 ? lds0 + STAGE : lds0;
            __builtin_amdgcn_sched_barrier(0);
#pragma unroll
            for (int m = 0; m < NM; ++m) {
                mfma_acc(acc[m / FQ][m % FQ], fp[0][m / FQ], fq[0][m % FQ]);
#pragma unroll
                for (int o = min(NR, m * NR * 3 / (NM * 2)); o < min(NR, (m + 1) * NR * 3 / (NM * 2)); ++o) read(o, 1, at);
                if (m % 2 == 0 && m / 2 < NDMA) look(m / 2);   // the rows of the DMAs behind the barrier
                __builtin_amdgcn_sched_barrier(0);
            }
            wait_vm<0>();   // the next stage is in place
            lds_barrier();  // for every wave, and every wave has read this one
            constexpr int NO = NR + NDMA;
#pragma unroll
            for (int m = 0; m < NM; ++m) {
                mfma_acc(acc[m / FQ][m % FQ], fp[1][m / FQ], fq[1][m % FQ]);
#pragma unroll
                for (int o = m * NO / NM; o < (m + 1) * NO / NM; ++o) {
                    const int rd = (o + 1) * NR / NO, rd0 = o * NR / NO;
                    if (rd > rd0) read(rd0, 0, nx);
                    else fetch(o - rd0, at);
                }
                __builtin_amdgcn_sched_barrier(0);
            }
            fetched();
            at = nx;
        }
        asm volatile("s_nop 15\n\ts_nop 15" ::: "memory");   // the last products end before their sums are read
#pragma unroll
        for (int i = 0; i < FP; ++i)
#pragma unroll
            for (int j = 0; j < FQ; ++j) asm volatile("" : "+a"(acc[i][j]));
        store_sums<T, F32, FP, FQ>(a, acc, ob, r0 + wq * 128, (col + t) * CN + wp * 128, lane);
#pragma unroll
        for (int i = 0; i < FP; ++i)
#pragma unroll
            for (int j = 0; j < FQ; ++j) acc[i][j] = f4{};
        asm volatile("s_nop 4" ::: "memory");
    }
    wait_vm<0>();
}

// Groups that mostly fit, matrices that fill 256 x 256 tiles, and a tile a CU.  Microseconds of bf16 gradients, tile kernels against
// k_gradients: 64 experts of 1024 x 2048 and 16 / 64 / 256 / 512 / 1024 pairs each 125 / 130 / 200 / 272 / 424 against 76 / 77 /
// 145 / 218 / 370; 8 experts 21 .. 61 against 16 .. 58; 4 experts (128 tiles) 12 .. 33 against 15 .. 54; 32 experts of 128 x 2048
// 12 .. 39 against 16 .. 52; 2048 tokens' pairs spread as 1 / rank^1.1 192 against 184.
static bool gradients(const MMArgs &a) {
    if (!a.egrp || !a.order || !a.vec || a.R <= 128 || a.N <= 128 || (a.accumulate && !a.out_f32) || a.ldp >= 1 << 30 || a.ldq >= 1 << 30 || a.ldo > 1 << 21) return false;
    const int64_t groups = std::max(1, std::min({a.max_active, a.n_expert, a.n_pairs}));
    return a.n_pairs <= PAIRS * groups && (int64_t) a.n_local * ((a.R + 255) / 256) * ((a.N + 255) / 256) >= 256;
}

template <typename T> static int launch_gradients(const MMArgs &a, hipStream_t s, const char *what) {
    const int64_t ncol = (a.N + 255) / 256, rows = (a.R + 255) / 256;
    const int64_t blocks = a.n_local * rows * ncol;
    // (8 tiles a block: as fast where the pairs are even, 330 for 187 us where they are spread as 1 / rank^1.1; 2 tiles: 172 for 152)
    const int nct = (int) std::min<int64_t>(std::clamp<int64_t>(blocks / 256, 1, 4), ncol);
    if (const int rc = check_blocks(what, blocks)) return rc;
    if (a.out_f32) k_gradients<T, true><<<(uint32_t) blocks, 256, 0, s>>>(a, nct);
    else k_gradients<T, false><<<(uint32_t) blocks, 256, 0, s>>>(a, nct);
    return check_launch(what);
}

// Gradients with fewer tiles than the card has CUs: the contraction is cut into parts, each a launch's worth of 128 x 128 tiles,
// whose fp32 sums are joined in order (no atomics: the same result every time).  Microseconds uncut / of 2, 4, 8, 16 parts (bf16):
// 8192 rows of 1024 x 1024 58 / 50, 36, 36, 50; of 512 x 512 54 / 46, 31, 22, 22; of 4096 x 1024 117 / 84, 93, 117, 187; 4096 rows of
// 2048 x 2048 66 / 52, 63, 90; 2048 rows of 1000 x 1032 19 / 23, 23, 27; 65536 rows of 64 x 2048 433 / 359, 192, 108, 69.
Parts dw_parts(int m, int n, int k) {
    constexpr TileCost cut{128, 128, 512, 0.66f, 0.75f, 0.95f, 5.0f};   // (a stage of parts reads less)
    MMArgs a{};
    a.R = n; a.N = k; a.K = m;
    if (n % 8 || k % 8) return Parts{1, m};   // rows that are not whole 16-byte pieces: k_mm_any, which goes through them uncut
    float least = tile_cost(TILES[cheapest(TILES, a, TN, false)], a, TN, false);
    Parts best{1, m};
    for (int p = 2; p <= 32; p *= 2) {
        const int len = (m / p / BK + 1) * BK, parts = len > 0 ? (m + len - 1) / len : 1;
        const double sums = (double) n * k * parts;
        if (parts < 2 || len < 4 * BK || sums > 1 << 26) break;   // (256 MB)
        MMArgs b = a;
        b.K = len;
        const float c = tile_cost(cut, b, TN, false, parts) + 5.0f + (float) (sums * 8 / 5e6);   // the join's launch, and its bytes at 5 MB / us
        if (c < least) { least = c; best = Parts{parts, len}; }
    }
    return best;
}

template <typename T> __global__ __launch_bounds__(256) void k_join(const MMArgs a) {
    const int64_t sums = (int64_t) a.R * a.N, pieces = sums / 4, all = pieces + (a.db ? a.R : 0);   // (N: a multiple of 8)
    for (int64_t i = (int64_t) blockIdx.x * 256 + threadIdx.x; i < all; i += (int64_t) gridDim.x * 256) {
        if (i < pieces) {
            union { f4 q; float v[4]; } s;
            s.q = f4{};
            for (int p = 0; p < a.parts; ++p) s.q += *(const f4 *) (a.part + p * sums + i * 4);
            const int64_t row = i * 4 / a.N, at = row * a.ldo + (i * 4 - row * a.N);
            if (a.accumulate) add_n<T, 4>(a.out, at, s.v, 4, a.out_f32, a.vec);
            put_n<T, 4>(a.out, at, s.v, 4, a.out_f32, a.vec);
        } else {
            const int64_t r = i - pieces;
            const float *d = a.part + a.parts * sums + r;
            float s = 0.0f;
            for (int p = 0; p < a.parts; ++p) s += d[(int64_t) p * a.R];
            a.db[r] = a.accumulate ? a.db[r] + s : s;
        }
    }
}

template <typename T> static int launch_parts(const MMArgs &a, hipStream_t s, const char *what) {
    MMArgs b = a;
    b.out = a.part; b.ldo = a.N; b.ostride = (int64_t) a.R * a.N; b.out_f32 = 1; b.accumulate = 0; b.vec = 1;
    if (a.db) b.db = a.part + a.parts * b.ostride;
    const int rc = launch_tile<T, TN, false, 128, 128, 2, 2, 2>(b, s, what);
    if (rc != HY_OK) return rc;
    const int64_t items = b.ostride / 4 + (a.db ? a.R : 0);
    k_join<T><<<(uint32_t) std::min<int64_t>((items + 255) / 256, 256 * 16), 256, 0, s>>>(a);
    return check_launch(what);
}

template <typename T> static int tiles(const MMArgs &a, hipStream_t s, const char *what) {
    if (a.parts > 1) return launch_parts<T>(a, s, what);
    if (gradients(a)) return launch_gradients<T>(a, s, what);
    switch (cheapest(TILES, a, TN, false)) {
    case 0: return launch_tile<T, TN, false, 256, 256, 2, 2, 2>(a, s, what);
    case 1: return launch_tile<T, TN, false, 128, 128, 2, 2, 2>(a, s, what);
    }
    return launch_tile<T, TN, false, 64, 128, 2, 2, 3>(a, s, what);
}
int launch_tiles_tn(int type, const MMArgs &a, hipStream_t s, const char *what) { return type == HY_BF16 ? tiles<bf16>(a, s, what) : tiles<f16>(a, s, what); }

} // namespace hy
