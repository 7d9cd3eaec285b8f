// C entries of what stands around the 16-bit products (include/hymoe.h): norms, routing with groups, low-rank adapters.
#include "hy_check16.h"
#include "hy_lora.cuh"
#include "hy_norm.cuh"

namespace hy {

int launch_route_groups(const float *logits, int64_t ls, int ne, const float *bias, bool softmax, int n_group, int top_group, int best, int k,
                        bool renorm, float scale, int *ids, float *wts, int nt, hipStream_t s);
int launch_route_groups_bwd(const float *logits, int64_t ls, int ne, bool softmax, const int *ids, int k, bool renorm, float scale, const float *dwts,
                            void *dlogits, int type, int64_t ldd, int nt, hipStream_t s);

static int check_type(const char *what, const char *name, int t) {
    if (t != HY_F32 && !type16(t)) { set_error("%s: %s type %d (HY_F32, HY_F16 or HY_BF16)", what, name, t); return HY_EUNSUPPORTED_TYPE; }
    return HY_OK;
}
static int bytes_of(int t) { return t == HY_F32 ? 4 : 2; }
// an array of fp32 or int32 values
static int check_vec(const char *what, const char *name, const void *p, bool need) {
    if (!p && need) { set_error("%s: %s is null", what, name); return HY_EINVAL; }
    if (misaligned(p, 4)) { set_error("%s: %s must be 4-byte aligned", what, name); return HY_EBAD_SHAPE; }
    return HY_OK;
}
// an output that takes an input's place must lie as it does: a row may only be written by those who have read it
static int check_place(const char *what, const char *name, const void *out, int64_t ldo, int out_bytes, const char *in_name, const void *in, int64_t ldi,
                       int in_bytes, int m) {
    if (!out || out != in || m < 1 || (out_bytes == in_bytes && (m == 1 || ldo == ldi))) return HY_OK;
    set_error("%s: %s takes the place of %s with other strides or another type", what, name, in_name);
    return HY_EBAD_SHAPE;
}
static int check_apart(const char *what, const char *one, const void *a, const char *other, const void *b) {
    if (!a || a != b) return HY_OK;
    set_error("%s: %s and %s are one place", what, one, other);
    return HY_EBAD_SHAPE;
}
static int check_norm_sizes(const char *what, int kind, int m, int n) {
    if (kind != HY_NORM_LAYER && kind != HY_NORM_RMS) { set_error("%s: kind %d", what, kind); return HY_EINVAL; }
    if (m < 0) { set_error("%s: %d rows", what, m); return HY_EINVAL; }
    if (m > HY_MM_MAX || n <= 0 || n > HY_NORM_MAX) { set_error("%s: m %d (up to 2^30), n %d (1 .. 2^22)", what, m, n); return HY_EBAD_SHAPE; }
    return HY_OK;
}
static int check_ws(const char *what, const void *ws, size_t ws_bytes, size_t need) {
    if (!need) return HY_OK;
    if (!ws || ws_bytes < need) { set_error("%s: workspace of %zu bytes, %zu needed", what, ws ? ws_bytes : (size_t) 0, need); return HY_EINVAL; }
    if (misaligned(ws, 16)) { set_error("%s: the workspace must be 16-byte aligned", what); return HY_EBAD_SHAPE; }
    return HY_OK;
}
static int check_route(const char *what, const float *logits, int64_t ls, int ne, int score, int k, int nt) {
    if (score != HY_SCORE_SOFTMAX && score != HY_SCORE_SIGMOID) { set_error("%s: score %d", what, score); return HY_EINVAL; }
    if (nt < 0) { set_error("%s: %d tokens", what, nt); return HY_EINVAL; }
    if (nt >= 1 << 24) { set_error("%s: %d tokens (a call takes less than 2^24)", what, nt); return HY_EBAD_SHAPE; }
    if (ne < 1 || ne > 1024) { set_error("%s: %d experts (1 .. 1024)", what, ne); return HY_EBAD_SHAPE; }
    if (k < 1 || k > 64) { set_error("%s: k = %d (1 .. 64)", what, k); return HY_EBAD_SHAPE; }
    if (nt == 0) return HY_OK;
    HY_TRY(check_vec(what, "logits", logits, true));
    if (ls < 0) { set_error("%s: %lld values between the rows of logits", what, (long long) ls); return HY_EBAD_SHAPE; }
    return HY_OK;
}

} // namespace hy

using namespace hy;

extern "C" {

int hy_norm(int kind, int x_type, const void *x, int64_t ldx, const void *add, int64_t ldadd, void *total, int64_t ldt, const float *w, const float *b,
            float eps, int m, int n, void *out, int out_type, int64_t ldo, float *out32, int64_t ldo32, float *mean, float *rstd, hipStream_t s) {
    const char *what = "hy_norm";
    HY_TRY(check_norm_sizes(what, kind, m, n));
    HY_TRY(check_type(what, "x", x_type));
    HY_TRY(check_type(what, "out", out_type));
    if (!out && !out32 && m) { set_error("%s: out and out32 are null", what); return HY_EINVAL; }
    if (!(eps >= 0.0f)) { set_error("%s: eps %g", what, (double) eps); return HY_EINVAL; }
    const int xb = bytes_of(x_type), ob = bytes_of(out_type);
    HY_TRY(check_mat(what, "x", x, ldx, m, n, xb, false));
    if (add) HY_TRY(check_mat(what, "add", add, ldadd, m, n, xb, false));
    if (total) HY_TRY(check_mat(what, "total", total, ldt, m, n, xb, true));
    if (out) HY_TRY(check_mat(what, "out", out, ldo, m, n, ob, true));
    if (out32) HY_TRY(check_mat(what, "out32", out32, ldo32, m, n, 4, true));
    HY_TRY(check_vec(what, "w", w, true));
    HY_TRY(check_vec(what, "b", b, false));
    HY_TRY(check_vec(what, "mean", mean, false));
    HY_TRY(check_vec(what, "rstd", rstd, false));
    if (m == 0) return HY_OK;
    HY_TRY(check_place(what, "total", total, ldt, xb, "x", x, ldx, xb, m));
    HY_TRY(check_place(what, "total", total, ldt, xb, "add", add, ldadd, xb, m));
    HY_TRY(check_place(what, "out", out, ldo, ob, "x", x, ldx, xb, m));
    HY_TRY(check_place(what, "out32", out32, ldo32, 4, "x", x, ldx, xb, m));
    HY_TRY(check_place(what, "out", out, ldo, ob, "add", add, ldadd, xb, m));
    HY_TRY(check_place(what, "out32", out32, ldo32, 4, "add", add, ldadd, xb, m));
    HY_TRY(check_apart(what, "total", total, "out", out));
    HY_TRY(check_apart(what, "total", total, "out32", out32));
    HY_TRY(check_apart(what, "out", out, "out32", out32));
    NormArgs a{};
    a.x = x; a.add = add; a.total = total; a.out = out; a.out32 = out32; a.w = w; a.b = b; a.mean = mean; a.rstd = rstd;
    a.ldx = ldx; a.lda = ldadd; a.ldt = ldt; a.ldo = ldo; a.ldo32 = ldo32; a.m = m; a.n = n; a.o_type = out_type; a.eps = eps;
    a.layer = kind == HY_NORM_LAYER;
    return launch_norm(x_type, a, s);
}

size_t hy_norm_bwd_ws_bytes(int m, int n) {
    if (m <= 0 || n <= 0 || n > HY_NORM_MAX) return 0;
    const int parts = norm_bwd_parts(m, n, false);
    return parts > 1 ? 2 * sizeof(float) * (size_t) parts * (size_t) n : 0;
}

int hy_norm_bwd(int kind, int x_type, const void *x, int64_t ldx, int dy_type, const void *dy, int64_t lddy, const float *w, const float *mean,
                const float *rstd, const void *resid, int64_t ldr, int m, int n, void *dx, int64_t lddx, float *dw, float *db, int accumulate,
                void *ws, size_t ws_bytes, hipStream_t s) {
    const char *what = "hy_norm_bwd";
    HY_TRY(check_norm_sizes(what, kind, m, n));
    HY_TRY(check_type(what, "x", x_type));
    HY_TRY(check_type(what, "dy", dy_type));
    const int xb = bytes_of(x_type), yb = bytes_of(dy_type);
    HY_TRY(check_mat(what, "x", x, ldx, m, n, xb, false));
    HY_TRY(check_mat(what, "dy", dy, lddy, m, n, yb, false));
    if (resid) HY_TRY(check_mat(what, "resid", resid, ldr, m, n, xb, false));
    HY_TRY(check_mat(what, "dx", dx, lddx, m, n, xb, true));
    HY_TRY(check_vec(what, "w", w, true));
    if (m) {   // (empty arrays have no address)
        HY_TRY(check_vec(what, "mean", mean, kind == HY_NORM_LAYER));
        HY_TRY(check_vec(what, "rstd", rstd, true));
    }
    HY_TRY(check_vec(what, "dw", dw, false));
    HY_TRY(check_vec(what, "db", db, false));
    if (db && kind == HY_NORM_RMS) { set_error("%s: an RMS norm has no b", what); return HY_EINVAL; }
    if (dw || db) HY_TRY(check_ws(what, ws, ws_bytes, hy_norm_bwd_ws_bytes(m, n)));
    HY_TRY(check_place(what, "dx", dx, lddx, xb, "x", x, ldx, xb, m));
    HY_TRY(check_place(what, "dx", dx, lddx, xb, "dy", dy, lddy, yb, m));
    HY_TRY(check_place(what, "dx", dx, lddx, xb, "resid", resid, ldr, xb, m));
    NormBwdArgs a{};
    a.x = x; a.dy = dy; a.resid = resid; a.dx = dx; a.w = w; a.mean = kind == HY_NORM_LAYER ? mean : nullptr; a.rstd = rstd; a.dw = dw; a.db = db;
    a.ldx = ldx; a.ldy = lddy; a.ldr = ldr; a.ldd = lddx; a.m = m; a.n = n; a.y_type = dy_type; a.accumulate = accumulate != 0;
    a.parts = m ? norm_bwd_parts(m, n, x_type == HY_F32) : 0;
    a.part = a.parts > 1 ? (float *) ws : nullptr;
    return launch_norm_bwd(x_type, kind == HY_NORM_LAYER, a, s);
}

int hy_moe_route_groups(const float *logits, int64_t ls, int n_expert, const float *bias, int score, int n_group, int top_group, int group_best,
                        int k, int renorm, float scale, int32_t *ids, float *wts, int nt, hipStream_t s) {
    const char *what = "hy_moe_route_groups";
    HY_TRY(check_route(what, logits, ls, n_expert, score, k, nt));
    if (n_group < 1 || n_group > 64 || n_expert % n_group) { set_error("%s: %d groups of %d experts (1 .. 64 equal ones)", what, n_group, n_expert); return HY_EBAD_SHAPE; }
    if (top_group < 1 || top_group > n_group) { set_error("%s: %d of %d groups", what, top_group, n_group); return HY_EBAD_SHAPE; }
    if (group_best != 1 && group_best != 2) { set_error("%s: groups by their %d best (1 or 2)", what, group_best); return HY_EINVAL; }
    const int gs = n_expert / n_group;
    if (top_group < n_group && gs < group_best) { set_error("%s: groups of %d by their %d best", what, gs, group_best); return HY_EBAD_SHAPE; }
    if (k > gs * top_group) { set_error("%s: k = %d of %d experts in %d groups", what, k, gs * top_group, top_group); return HY_EBAD_SHAPE; }
    if (nt == 0) return HY_OK;
    HY_TRY(check_vec(what, "bias", bias, false));
    HY_TRY(check_vec(what, "ids", ids, true));
    HY_TRY(check_vec(what, "wts", wts, true));
    return launch_route_groups(logits, ls, n_expert, bias, score == HY_SCORE_SOFTMAX, n_group, top_group, group_best, k, renorm != 0, scale, ids, wts, nt, s);
}

int hy_moe_route_groups_bwd(const float *logits, int64_t ls, int n_expert, int score, const int32_t *ids, int k, int renorm, float scale,
                            const float *dwts, void *dlogits, int type, int64_t ldd, int nt, hipStream_t s) {
    const char *what = "hy_moe_route_groups_bwd";
    HY_TRY(check_route(what, logits, ls, n_expert, score, k, nt));
    HY_TRY(check_type(what, "dlogits", type));
    if (nt == 0) return HY_OK;
    HY_TRY(check_vec(what, "ids", ids, true));
    HY_TRY(check_vec(what, "dwts", dwts, true));
    HY_TRY(check_mat(what, "dlogits", dlogits, ldd, nt, n_expert, bytes_of(type), true));
    HY_TRY(check_place(what, "dlogits", dlogits, ldd, bytes_of(type), "logits", logits, ls, 4, nt));
    return launch_route_groups_bwd(logits, ls, n_expert, score == HY_SCORE_SOFTMAX, ids, k, renorm != 0, scale, dwts, dlogits, type, ldd, nt, s);
}

size_t hy_lora_ws_bytes(int m, int r, int k) {
    if (m <= 0 || r <= 0 || k <= 0 || m > HY_MM_MAX || r > HY_LORA_MAX_RANK || k > HY_MM_MAX) return 0;
    return sizeof(float) * (size_t) lora_cut(m, k).splits * (size_t) m * (size_t) r;
}

int hy_lora(int type, const void *A, const void *B, const float *scale, int n_local, int r, int k, int n, const void *x, int64_t ldx, int m,
            const int32_t *ids, const void *resid, int64_t ldr, void *out, int out_type, int64_t ldo, void *ws, size_t ws_bytes, hipStream_t s) {
    const char *what = "hy_lora";
    HY_TRY(check_sizes(what, type, m, n, k));
    HY_TRY(check_out_type(what, type, out_type));
    if (n_local < 1 || n_local > HY_MM_MAX) { set_error("%s: %d adapters", what, n_local); return HY_EINVAL; }
    if (r < 1 || r > HY_LORA_MAX_RANK) { set_error("%s: rank %d (1 .. %d)", what, r, HY_LORA_MAX_RANK); return HY_EBAD_SHAPE; }
    const int ob = out_type == HY_F32 ? 4 : 2;
    HY_TRY(check_mat(what, "A", A, k, r, k, 2, false));
    HY_TRY(check_mat(what, "B", B, r, n, r, 2, false));
    HY_TRY(check_vec(what, "scale", scale, false));
    HY_TRY(check_mat(what, "x", x, ldx, m, k, 2, false));
    HY_TRY(check_mat(what, "out", out, ldo, m, n, ob, true));
    if (resid) HY_TRY(check_mat(what, "resid", resid, ldr, m, n, ob, false));
    if (m == 0) return HY_OK;
    HY_TRY(check_vec(what, "ids", ids, true));
    HY_TRY(check_ws(what, ws, ws_bytes, hy_lora_ws_bytes(m, r, k)));
    const LoraCut cut = lora_cut(m, k);
    HY_TRY(check_blocks(what, (int64_t) ((m + 15) / 16) * ((n + 255) / 256)));
    if (ldo > HY_LORA_MAX_STRIDE || (resid && ldr > HY_LORA_MAX_STRIDE) || n > HY_LORA_MAX_STRIDE) { set_error("%s: rows of out or resid more than 2^22 values apart", what); return HY_EBAD_SHAPE; }
    HY_TRY(check_place(what, "out", out, ldo, ob, "resid", resid, ldr, ob, m));
    LoraArgs a{};
    a.A = A; a.B = B; a.x = x; a.scale = scale; a.ids = ids; a.resid = resid; a.out = out; a.low = (float *) ws;
    a.ldx = ldx; a.ldr = ldr; a.ldo = ldo; a.m = m; a.n = n; a.k = k; a.r = r; a.n_local = n_local;
    a.splits = cut.splits; a.klen = cut.klen; a.out_f32 = out_type == HY_F32;
    return launch_lora(type, a, s);
}

} // extern "C"
