// Routing with groups of experts, and its gradient.
//
// s = softmax(l) or sigmoid(l);  c = s + bias;  a group's worth is the sum of its `best` largest c;  of the top_group best groups
// the k experts with the largest c;  weights s scale, renormalised over the chosen on request.  Ties go to the lower index.
// The choice is that of the formula in 64 bits: scores, their sum, the worths and the weights are doubles (vector double
// arithmetic runs at the rate of single here), so two experts whose scores differ by less than a single holds still come in
// the formula's order.  One wave a token; bound by latency, and from a few thousand tokens on by the arithmetic.
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
__device__ __forceinline__ double wave_sum_d(double v) {
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) v += shfl_xor_d(v, o);
    return v;
}
// a double as an unsigned key of the same order, above 0 (-0 as +0); 0 is left for what may not be chosen
__device__ __forceinline__ uint64_t order_key_d(double d) {
    const uint64_t u = (uint64_t) __double_as_longlong(d == 0.0 ? 0.0 : d);
    return (u >> 63) ? ~u : (u | 1ull << 63);
}
__device__ __forceinline__ double sigmoid_d(double x) { return 1.0 / (1.0 + exp(-x)); }

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
// are left.  The k-th largest of the lanes' maxima, taken on the keys' upper halves, bounds the k-th key from below; what lies at
// or above it (usually little more than k keys) is gathered in index order and ranked by counting.  More than 64 of them
// (many equal scores): one expert after the other.
template <int V> __device__ __forceinline__ int wave_topk_d(uint64_t (&key)[V], int k, uint64_t *c_key, int *c_idx, int *r_idx) {
    const int lane = threadIdx.x & 63;
    uint32_t lmax = 0;
#pragma unroll
    for (int i = 0; i < V; ++i) { const uint32_t h = (uint32_t) (key[i] >> 32); lmax = h > lmax ? h : lmax; }
    uint32_t th = 1;   // (a key's upper half is 0 for what may not be chosen alone: every double but NaN is above 2^32)
    {
        const uint32_t lm[1] = {lmax};
        const bool on[1] = {lmax != 0};
        const uint32_t t = wave_kth_key<1>(lm, on, k);
        th = t > th ? t : th;
    }
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

template <int V> __global__ __launch_bounds__(64 * RG_WAVES) void k_route_groups(const RouteArgs a) {
    __shared__ double s_c[RG_WAVES][64 * V];
    __shared__ uint64_t s_key[RG_WAVES][64];
    __shared__ int s_idx[RG_WAVES][64], s_rank[RG_WAVES][64];
    const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63, t = blockIdx.x * RG_WAVES + wave;
    if (t >= a.nt) return;   // (no block barrier below)
    const float *l = a.logits + (int64_t) t * a.ls;
    float x[V];
    load_logits<V>(l, a.ne, x);
    double c[V];
    double top = 0.0, sum = 0.0;
    if (a.softmax) {
        float mf = x[0];
#pragma unroll
        for (int i = 1; i < V; ++i) mf = fmaxf(mf, x[i]);
        top = (double) wave_max(mf);
#pragma unroll
        for (int i = 0; i < V; ++i) { c[i] = lane + 64 * i < a.ne ? exp((double) x[i] - top) : 0.0; sum += c[i]; }
        sum = wave_sum_d(sum);
#pragma unroll
        for (int i = 0; i < V; ++i) c[i] = c[i] / sum;
    } else {
#pragma unroll
        for (int i = 0; i < V; ++i) c[i] = sigmoid_d((double) x[i]);
    }
    // what may not be chosen is -inf from here on: experts behind the last, logits of -inf, NaN anywhere
#pragma unroll
    for (int i = 0; i < V; ++i) {
        const int e = lane + 64 * i;
        if (a.bias && e < a.ne) c[i] += (double) a.bias[e];
        if (!(e < a.ne && x[i] > -__builtin_huge_valf() && c[i] > -D_INF)) c[i] = -D_INF;
    }
    uint64_t keep = ~0ull;
    if (a.top_group < a.n_group) {
        double *sc = s_c[wave];
#pragma unroll
        for (int i = 0; i < V; ++i) sc[lane + 64 * i] = c[i];
        wave_lds_sync();
        const int lpg = 1 << a.lsh, g = lane >> a.lsh, q = lane & (lpg - 1);
        double b1 = -D_INF, b2 = -D_INF;
        if (g < a.n_group) {
            for (int j = q; j < a.gs; j += lpg) {
                const double v = sc[g * a.gs + j];
                if (v > b1) { b2 = b1; b1 = v; } else if (v > b2) b2 = v;
            }
        }
        for (int o = 1; o < lpg; o <<= 1) {
            const double o1 = shfl_xor_d(b1, o), o2 = shfl_xor_d(b2, o);
            if (o1 > b1) { b2 = b1 > o2 ? b1 : o2; b1 = o1; } else b2 = b2 > o1 ? b2 : o1;
        }
        const double worth = a.best == 1 ? b1 : b2 > -D_INF ? b1 + b2 : -D_INF;
        int rank = 0;
        for (int i = 0; i < a.n_group; ++i) {
            const double w = readlane_d(worth, i << a.lsh);
            rank += (w > worth) | ((w == worth) & (i < g));
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
    const double z = on ? (double) l[e] : -D_INF;
    double w;
    if (a.softmax) {
        if (a.renorm) {   // over the largest chosen logit: no weight's exponential is lost beside one that was not chosen
            const float zm = wave_max(on ? (float) z : -__builtin_huge_valf());
            w = on ? exp(z - (double) zm) : 0.0;
        } else w = on ? exp(z - top) / sum : 0.0;
    } else w = on ? sigmoid_d(z) : 0.0;
    if (a.renorm) {
        const double S = wave_sum_d(w);
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
            for (int i = 0; i < V; ++i) { p[i] = lane + 64 * i < a.ne ? exp((double) x[i] - m) : 0.0; sum += p[i]; }
            sum = wave_sum_d(sum);
            const double dot = wave_sum_d(on ? exp((double) zf - m) * f : 0.0) / sum;
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
            for (int i = 0; i < V; ++i) d[i] = (float) (p[i] / sum * (fe[i] - dot));
        } else {
            double v, keep = 1.0;   // keep: 1 - s of a sigmoid
            const double zm = (double) wave_max(zf);
            if (a.softmax) v = on ? exp((double) zf - zm) : 0.0;
            else {
                const double ez = exp(-fabs((double) zf)), hi = 1.0 / (1.0 + ez), lo = ez * hi;   // sigmoid of |z| and of -|z|
                v = on ? (zf >= 0.0f ? hi : zf < 0.0f ? lo : (double) zf) : 0.0;   // (NaN stays)
                keep = zf >= 0.0f ? lo : hi;
            }
            if (a.renorm) {
                const double S = wave_sum_d(v);
                v = S == 0.0 ? 0.0 : v / S;
                dz = v * keep * (f - wave_sum_d(v * f));
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
    const dim3 grid((nt + RG_WAVES - 1) / RG_WAVES), block(64 * RG_WAVES);
    const int V = (ne + 63) / 64;
    if (V <= 1) k_route_groups<1><<<grid, block, 0, s>>>(a);
    else if (V <= 2) k_route_groups<2><<<grid, block, 0, s>>>(a);
    else if (V <= 4) k_route_groups<4><<<grid, block, 0, s>>>(a);
    else if (V <= 8) k_route_groups<8><<<grid, block, 0, s>>>(a);
    else k_route_groups<16><<<grid, block, 0, s>>>(a);
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
