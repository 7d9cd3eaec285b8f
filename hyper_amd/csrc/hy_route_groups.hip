// Routing with groups of experts, and its gradient.
//
// s = softmax(l) or sigmoid(l);  c = s + bias;  a group's worth is the sum of its `best` largest c;  of the top_group best groups
// the k experts with the largest c;  weights s scale, renormalised over the chosen on request.  Ties go to the lower index.
// The choice is that of the formula in 64 bits: scores, their sum, the worths and the weights are doubles (vector double
// arithmetic runs at the rate of single here), so two experts whose scores differ by less than a single holds still come in
// the formula's order.  A score is off by up to 4 2^-53 of itself (exp, its sum, the reciprocal), bias and worth round by 2^-53:
// only what lies closer than that may change places.  One wave a token; bound by latency (one token, 384 experts in 8 groups: 5.2 us), and from
// a few thousand tokens on by the arithmetic (8192 tokens, 256 experts: 13 us, 571 vector instructions each).
#include "hy_routing.cuh"
#include "hy_mm16.cuh"

#include <algorithm>

namespace hy {

constexpr double D_INF = __builtin_huge_val();

__device__ __forceinline__ double shfl_xor_d(double v, int o) {
    const uint64_t u = (uint64_t) __double_as_longlong(v);
    const uint32_t lo = (uint32_t) __shfl_xor((int) (uint32_t) u, o), hi = (uint32_t) __shfl_xor((int) (uint32_t) (u >> 32), o);
    return __longlong_as_double((long long) ((uint64_t) hi << 32 | lo));
}
__device__ __forceinline__ double readlane_d(double v, int l) {
    const uint64_t u = (uint64_t) __double_as_longlong(v);
    const uint32_t lo = (uint32_t) __builtin_amdgcn_readlane((int) (uint32_t) u, l), hi = (uint32_t) __builtin_amdgcn_readlane((int) (uint32_t) (u >> 32), l);
    return __longlong_as_double((long long) ((uint64_t) hi << 32 | lo));
}
__device__ __forceinline__ double shfl_d(double v, int l) {
    const uint64_t u = (uint64_t) __double_as_longlong(v);
    const uint32_t lo = (uint32_t) __shfl((int) (uint32_t) u, l), hi = (uint32_t) __shfl((int) (uint32_t) (u >> 32), l);
    return __longlong_as_double((long long) ((uint64_t) hi << 32 | lo));
}
__device__ __forceinline__ double wave_sum_d(double v) {
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) v += shfl_xor_d(v, o);
    return v;
}
// the sum of the first k lanes' values in these lanes (the others hold zeros)
__device__ __forceinline__ double chosen_sum_d(double v, int k) {
    for (int o = 1; o < k; o <<= 1) v += shfl_xor_d(v, o);
    return v;
}
// a double as an unsigned key of the same order, above 0 (-0 as +0); 0 is left for what may not be chosen
__device__ __forceinline__ uint64_t order_key_d(double d) {
    const uint64_t u = (uint64_t) __double_as_longlong(d == 0.0 ? 0.0 : d);
    return (u >> 63) ? ~u : (u | 1ull << 63);
}
// exp(x) for x <= 0 (0 below -745, where the nearest value is) by Cody and Waite: x = n ln 2 + r, ln 2 in two parts whose first has 21 zero
// bits (n times it is exact), exp(r) by its Taylor polynomial, 2^n as a shift of the exponent.  |r| <= 0.3466: the first term
// left out, r^14 / 14!, is 4e-18.  NaN stays.
__device__ __forceinline__ double exp_neg_d(double x) {
    const double n = __builtin_rint(x * 1.4426950408889634);
    double r = __builtin_fma(n, -0.69314718036912382, x);
    r = __builtin_fma(n, -1.9082149292705877e-10, r);
    double p = 1.6059043836821613e-10;
    p = __builtin_fma(p, r, 2.08767569878681e-9);
    p = __builtin_fma(p, r, 2.505210838544172e-8);
    p = __builtin_fma(p, r, 2.755731922398589e-7);
    p = __builtin_fma(p, r, 2.7557319223985893e-6);
    p = __builtin_fma(p, r, 2.48015873015873e-5);
    p = __builtin_fma(p, r, 1.984126984126984e-4);
    p = __builtin_fma(p, r, 1.3888888888888889e-3);
    p = __builtin_fma(p, r, 8.333333333333333e-3);
    p = __builtin_fma(p, r, 4.1666666666666664e-2);
    p = __builtin_fma(p, r, 1.6666666666666666e-1);
    p = __builtin_fma(p, r, 0.5);
    p = __builtin_fma(p, r, 1.0);
    p = __builtin_fma(p, r, 1.0);
    const double v = __builtin_amdgcn_ldexp(p, (int) n);
    return x < -745.2 ? 0.0 : v;
}
// 1 / d for d in [1, 2] and for a softmax's sum in [1, 1024]: Newton's iteration from the hardware's estimate
__device__ __forceinline__ double rcp_d(double d) {
    double y = __builtin_amdgcn_rcp(d);
    y = __builtin_fma(__builtin_fma(-d, y, 1.0), y, y);
    return __builtin_fma(__builtin_fma(-d, y, 1.0), y, y);
}
// sigmoid(x) and 1 - it, from exp(-|x|): neither end overflows or cancels.  NaN stays.
__device__ __forceinline__ void sigmoid_d(double x, double &s, double &rest) {
    const double e = exp_neg_d(-__builtin_fabs(x)), big = rcp_d(1.0 + e), small = e * big;
    s = x < 0.0 ? small : big;
    rest = x < 0.0 ? big : small;
}
__device__ __forceinline__ double sigmoid_d(double x) {
    double s, rest;
    sigmoid_d(x, s, rest);
    return s;
}

struct RouteArgs {
    const float *logits, *bias;
    int *ids;
    float *wts;
    int64_t ls;
    int nt, ne, k, n_group, top_group, best, gs, lsh;   // experts of a group; lsh: 2^lsh lanes search one
    double scale;
    bool softmax, renorm;
};

// Top k of the keys (element lane + 64 i in slot i; 0: not to be chosen): lane r < k gets the index of rank r, or -1 where fewer
// are left.  The k-th largest of the lanes' maxima bounds the k-th key from below; what lies at
// or above it (usually little more than k keys) is gathered in index order and ranked by counting.  More than 64 of them
// (many equal scores): one expert after the other.
template <int V> __device__ __forceinline__ int wave_topk_d(uint64_t (&key)[V], int k, uint64_t *c_key, int *c_idx, int *r_idx) {
    const int lane = threadIdx.x & 63;
    uint32_t lmax = 0;
#pragma unroll
    for (int i = 0; i < V; ++i) { const uint32_t h = (uint32_t) (key[i] >> 32); lmax = h > lmax ? h : lmax; }
    // The bound's upper 20 bits (an eighth of a binary place in 2^-8 steps), bit by bit; below, zeros: a few keys more to rank
    uint32_t th = 0;
    for (int b = 31; b >= 12; --b) {
        const uint32_t c = th | 1u << b;
        if (__popcll(__ballot(lmax >= c)) >= k) th = c;   // wave-uniform
    }
    th = th ? th : 1;   // (a key's upper half is 0 for what may not be chosen alone: every double but NaN is above 2^32)
    int n_c = 0;
#pragma unroll
    for (int i = 0; i < V; ++i) n_c += __popcll(__ballot((uint32_t) (key[i] >> 32) >= th));
    int out = -1;
    if (n_c <= 64) {
        n_c = 0;
#pragma unroll
        for (int i = 0; i < V; ++i) {
            const bool take = (uint32_t) (key[i] >> 32) >= th;
            const uint64_t m = __ballot(take);
            if (take) {
                const int at = n_c + lanes_below(m);
                c_key[at] = key[i];
                c_idx[at] = lane + 64 * i;
            }
            n_c += __popcll(m);
        }
        wave_lds_sync();
        const uint64_t mine = lane < n_c ? c_key[lane] : 0;
        const int my_idx = lane < n_c ? c_idx[lane] : -1;
        int rank = 0;
        for (int m = 0; m < n_c; ++m) {
            const uint32_t lo = (uint32_t) __builtin_amdgcn_readlane((int) (uint32_t) mine, m), hi = (uint32_t) __builtin_amdgcn_readlane((int) (uint32_t) (mine >> 32), m);
            const uint64_t km = (uint64_t) hi << 32 | lo;
            rank += (km > mine) | ((km == mine) & (m < lane));
        }
        r_idx[lane] = -1;
        wave_lds_sync();
        if (lane < n_c && rank < k) r_idx[rank] = my_idx;
        wave_lds_sync();
        out = r_idx[lane];
    } else {
        for (int r = 0; r < k; ++r) {
            uint64_t bk = 0;
            int bi = 0x7fffffff;
#pragma unroll
            for (int i = 0; i < V; ++i) if (key[i] > bk) { bk = key[i]; bi = lane + 64 * i; }
#pragma unroll
            for (int o = 1; o < 64; o <<= 1) {
                const uint32_t lo = (uint32_t) __shfl_xor((int) (uint32_t) bk, o), hi = (uint32_t) __shfl_xor((int) (uint32_t) (bk >> 32), o);
                const int oi = __shfl_xor(bi, o);
                const uint64_t ok = (uint64_t) hi << 32 | lo;
                if (ok > bk || (ok == bk && oi < bi)) { bk = ok; bi = oi; }
            }
            if (bk == 0) break;   // none left (the same in every lane)
            if (lane == r) out = bi;
#pragma unroll
            for (int i = 0; i < V; ++i) if (lane + 64 * i == bi) key[i] = 0;
        }
    }
    return out;
}

constexpr int RG_WAVES = 4;   // tokens a block
__host__ __device__ constexpr int rg_waves(int V) { return V > 8 ? 2 : RG_WAVES; }   // (the scores' LDS)

template <int V> __global__ __launch_bounds__(64 * rg_waves(V)) void k_route_groups(const RouteArgs a) {
    constexpr int RG_WAVES = rg_waves(V);
    __shared__ double s_score[RG_WAVES][64 * V], s_c[RG_WAVES][64 * V];
    __shared__ uint64_t s_key[RG_WAVES][64];
    __shared__ int s_idx[RG_WAVES][64], s_rank[RG_WAVES][64];
    const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63, t = blockIdx.x * RG_WAVES + wave;
    if (t >= a.nt) return;   // (no block barrier below)
    const float *l = a.logits + (int64_t) t * a.ls;
    float x[V];
    load_logits<V>(l, a.ne, x);
    float bias[V];   // (loaded with the logits, not behind the scores)
#pragma unroll
    for (int i = 0; i < V; ++i) bias[i] = a.bias && lane + 64 * i < a.ne ? a.bias[lane + 64 * i] : 0.0f;
    double c[V];
    double top = 0.0, sum = 0.0;   // sum: then its reciprocal
    if (a.softmax) {
        float mf = x[0];
#pragma unroll
        for (int i = 1; i < V; ++i) mf = fmaxf(mf, x[i]);
        top = (double) wave_max(mf);
#pragma unroll
        for (int i = 0; i < V; ++i) { c[i] = lane + 64 * i < a.ne ? exp_neg_d((double) x[i] - top) : 0.0; sum += c[i]; }
        sum = rcp_d(wave_sum_d(sum));
#pragma unroll
        for (int i = 0; i < V; ++i) c[i] *= sum;
    } else {
#pragma unroll
        for (int i = 0; i < V; ++i) c[i] = sigmoid_d((double) x[i]);
    }
#pragma unroll
    for (int i = 0; i < V; ++i) s_score[wave][lane + 64 * i] = c[i];
    // what may not be chosen is -inf from here on: experts behind the last, logits of -inf, NaN anywhere
#pragma unroll
    for (int i = 0; i < V; ++i) {
        const int e = lane + 64 * i;
        c[i] += (double) bias[i];
        if (!(e < a.ne && x[i] > -__builtin_huge_valf() && c[i] > -D_INF)) c[i] = -D_INF;
    }
    uint64_t keep = ~0ull;
    if (a.top_group < a.n_group) {
        double *sc = s_c[wave];
#pragma unroll
        for (int i = 0; i < V; ++i) sc[lane + 64 * i] = c[i];
        wave_lds_sync();
        const int lpg = 1 << a.lsh, g = lane >> a.lsh, q = lane & (lpg - 1);
        double b1 = -D_INF, b2 = -D_INF;   // the two largest so far (no NaN among them)
        if (g < a.n_group) {
#pragma unroll 4
            for (int j = q; j < a.gs; j += lpg) {
                const double v = sc[g * a.gs + j];
                b2 = __builtin_fmax(b2, __builtin_fmin(b1, v));
                b1 = __builtin_fmax(b1, v);
            }
        }
        for (int o = 1; o < lpg; o <<= 1) {
            const double o1 = shfl_xor_d(b1, o), o2 = shfl_xor_d(b2, o);
            b2 = __builtin_fmax(__builtin_fmin(b1, o1), __builtin_fmax(b2, o2));
            b1 = __builtin_fmax(b1, o1);
        }
        const double worth = a.best == 1 ? b1 : b2 > -D_INF ? b1 + b2 : -D_INF;
        // the group's rank: each of its lanes compares it with other groups
        int rank = 0;
        for (int i = 0; i < a.n_group; i += lpg) {
            const double w = shfl_d(worth, ((i + q) << a.lsh) & 63);
            const uint64_t before = __ballot(i + q < a.n_group && (w > worth || (w == worth && i + q < g)));
            rank += __popcll(before >> (g << a.lsh) & (lpg == 64 ? ~0ull : (1ull << lpg) - 1));
        }
        keep = __ballot(q == 0 && g < a.n_group && rank < a.top_group && worth > -D_INF);
    }
    uint64_t key[V];
    const float per = 1.0f / (float) a.gs;
#pragma unroll
    for (int i = 0; i < V; ++i) {
        const int g = (int) (((float) (lane + 64 * i) + 0.5f) * per);   // e / gs: at least 0.5 / gs from the next whole number
        const bool in = a.top_group >= a.n_group || (keep >> ((g << a.lsh) & 63) & 1);
        key[i] = in && c[i] > -D_INF ? order_key_d(c[i]) : 0;
    }
    const int e = wave_topk_d<V>(key, a.k, s_key[wave], s_idx[wave], s_rank[wave]);
    const bool on = lane < a.k && e >= 0;
    wave_lds_sync();
    double w = on ? s_score[wave][e] : 0.0;
    if (a.softmax && a.renorm) {   // over the largest chosen logit: no weight's exponential is lost beside one that was not chosen
        const float z = on ? l[e] : -__builtin_huge_valf(), zm = wave_max(z);
        w = on ? exp_neg_d((double) z - (double) zm) : 0.0;
    }
    if (a.renorm) {
        const double S = chosen_sum_d(w, a.k);
        w = S > 0.0 ? w / S : 0.0;
    }
    if (lane < a.k) {
        a.ids[(int64_t) t * a.k + lane] = e;
        a.wts[(int64_t) t * a.k + lane] = (float) (w * a.scale);
    }
}

// ------------------------------------------------------------------ gradient

// From dw of the weights w = scale s (or scale s / S, S the sum of the chosen s), with f_r = dw_r scale:
//   softmax, renormalised   w is a softmax of the chosen logits:  dl_r = v_r (f_r - sum v f),  v = s / S
//   sigmoid, renormalised   dl_r = (1 - s_r) v_r (f_r - sum v f)
//   sigmoid                 dl_r = s_r (1 - s_r) f_r
//   softmax                 dl_e = s_e (f_e - sum s f) for every expert, f_e = 0 where not chosen
// and 0 elsewhere.  A chosen logit is read alone unless the sum runs over all; the row is written in one pass, each chosen
// expert's value picked by comparing indices (an expert that ids names twice gets both).
struct RouteBwdArgs {
    const float *logits, *dwts;
    const int *ids;
    void *out;
    int64_t ls, ldo;
    int nt, ne, k;
    double scale;
    bool softmax, renorm;
};
template <int V, typename T> __global__ __launch_bounds__(64 * RG_WAVES) void k_route_groups_bwd(const RouteBwdArgs a) {
    const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63, t = blockIdx.x * RG_WAVES + wave;
    if (t >= a.nt) return;
    const float *l = a.logits + (int64_t) t * a.ls;
    const int id = lane < a.k ? a.ids[(int64_t) t * a.k + lane] : -1;
    const bool on = (uint32_t) id < (uint32_t) a.ne;
    const uint64_t any = __ballot(on);
    const float zf = on ? l[id] : -__builtin_huge_valf();
    const double f = on ? (double) a.dwts[(int64_t) t * a.k + lane] * a.scale : 0.0;
    float d[V];
#pragma unroll
    for (int i = 0; i < V; ++i) d[i] = 0.0f;
    double dz = 0.0;
    if (any) {
        if (a.softmax && !a.renorm) {
            float x[V];
            load_logits<V>(l, a.ne, x);
            float mf = x[0];
#pragma unroll
            for (int i = 1; i < V; ++i) mf = fmaxf(mf, x[i]);
            const double m = (double) wave_max(mf);
            double p[V], sum = 0.0;
#pragma unroll
            for (int i = 0; i < V; ++i) { p[i] = lane + 64 * i < a.ne ? exp_neg_d((double) x[i] - m) : 0.0; sum += p[i]; }
            sum = rcp_d(wave_sum_d(sum));
            double dot = chosen_sum_d(on ? exp_neg_d((double) zf - m) * f : 0.0, a.k) * sum;
            dot = readlane_d(dot, 0);
            double fe[V];
#pragma unroll
            for (int i = 0; i < V; ++i) fe[i] = 0.0;
            for (int r = 0; r < a.k; ++r) {
                const int e = __builtin_amdgcn_readlane(id, r);
                const double fr = readlane_d(f, r);
#pragma unroll
                for (int i = 0; i < V; ++i) if (lane + 64 * i == e) fe[i] += fr;
            }
#pragma unroll
            for (int i = 0; i < V; ++i) d[i] = (float) (p[i] * sum * (fe[i] - dot));
        } else {
            double v, keep = 1.0;   // keep: 1 - s of a sigmoid
            const double zm = (double) wave_max(zf);
            if (a.softmax) v = on ? exp_neg_d((double) zf - zm) : 0.0;
            else {
                sigmoid_d((double) zf, v, keep);
                v = on ? v : 0.0;
            }
            if (a.renorm) {
                const double S = chosen_sum_d(v, a.k);
                v = S == 0.0 ? 0.0 : v / S;
                dz = v * keep * (f - chosen_sum_d(v * f, a.k));
            } else dz = v * keep * f;
            for (int r = 0; r < a.k; ++r) {
                const int e = __builtin_amdgcn_readlane(id, r);
                const float dr = readlane_f((float) dz, r);
#pragma unroll
                for (int i = 0; i < V; ++i) if (lane + 64 * i == e) d[i] += dr;
            }
        }
    }
    T *o = (T *) a.out + (int64_t) t * a.ldo;
#pragma unroll
    for (int i = 0; i < V; ++i) if (lane + 64 * i < a.ne) o[lane + 64 * i] = (T) d[i];
}

int launch_route_groups(const float *logits, int64_t ls, int ne, const float *bias, bool softmax, int n_group, int top_group, int best, int k,
                        bool renorm, float scale, int *ids, float *wts, int nt, hipStream_t s) {
    RouteArgs a{};
    a.logits = logits; a.bias = bias; a.ids = ids; a.wts = wts; a.ls = ls; a.nt = nt; a.ne = ne; a.k = k;
    a.n_group = n_group; a.top_group = top_group; a.best = best; a.gs = ne / n_group;
    while (2 * n_group << a.lsh <= 64) ++a.lsh;
    a.scale = scale; a.softmax = softmax; a.renorm = renorm;
    const int V = (ne + 63) / 64;
#define HY_RG(V) k_route_groups<V><<<(nt + rg_waves(V) - 1) / rg_waves(V), 64 * rg_waves(V), 0, s>>>(a)
    if (V <= 1) HY_RG(1);
    else if (V <= 2) HY_RG(2);
    else if (V <= 4) HY_RG(4);
    else if (V <= 6) HY_RG(6);
    else if (V <= 8) HY_RG(8);
    else HY_RG(16);
#undef HY_RG
    return check_launch("hy_moe_route_groups");
}
template <int V> static void launch_bwd_v(int type, const RouteBwdArgs &a, hipStream_t s) {
    const dim3 grid((a.nt + RG_WAVES - 1) / RG_WAVES), block(64 * RG_WAVES);
    if (type == HY_F32) k_route_groups_bwd<V, float><<<grid, block, 0, s>>>(a);
    else if (type == HY_BF16) k_route_groups_bwd<V, bf16><<<grid, block, 0, s>>>(a);
    else k_route_groups_bwd<V, f16><<<grid, block, 0, s>>>(a);
}
int launch_route_groups_bwd(const float *logits, int64_t ls, int ne, bool softmax, const int *ids, int k, bool renorm, float scale, const float *dwts,
                            void *dlogits, int type, int64_t ldd, int nt, hipStream_t s) {
    RouteBwdArgs a{};
    a.logits = logits; a.dwts = dwts; a.ids = ids; a.out = dlogits; a.ls = ls; a.ldo = ldd; a.nt = nt; a.ne = ne; a.k = k;
    a.scale = scale; a.softmax = softmax; a.renorm = renorm;
    const int V = (ne + 63) / 64;
    if (V <= 1) launch_bwd_v<1>(type, a, s);
    else if (V <= 2) launch_bwd_v<2>(type, a, s);
    else if (V <= 4) launch_bwd_v<4>(type, a, s);
    else if (V <= 8) launch_bwd_v<8>(type, a, s);
    else launch_bwd_v<16>(type, a, s);
    return check_launch("hy_moe_route_groups_bwd");
}

} // namespace hy
