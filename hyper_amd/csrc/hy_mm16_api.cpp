// C entries of the 16-bit matrix products (include/hymoe.h): argument checks and dispatch.
#include "hy_mm16.cuh"

namespace hy {

static bool type16(int t) { return t == HY_F16 || t == HY_BF16; }
static bool misaligned(const void *p, size_t a) { return ((uintptr_t) p & (a - 1)) != 0; }

// a matrix of `rows` x `cols` elements of `bytes` each whose rows lie `ld` elements apart; out: written
static int check_mat(const char *what, const char *name, const void *p, int64_t ld, int rows, int cols, int bytes, bool out) {
    if (!rows) return HY_OK;   // an empty matrix may have no address
    if (!p) { set_error("%s: %s is null", what, name); return HY_EINVAL; }
    if (misaligned(p, bytes)) { set_error("%s: %s is not aligned to its %d-byte values", what, name, bytes); return HY_EBAD_SHAPE; }
    if (ld < 0 || (out && rows > 1 && ld < cols)) { set_error("%s: %lld elements between the rows of %s (%d values)", what, (long long) ld, name, cols); return HY_EBAD_SHAPE; }
    return HY_OK;
}
static int check_sizes(const char *what, int type, int m, int n, int k) {
    if (!type16(type)) { set_error("%s: type %d (HY_F16 or HY_BF16)", what, type); return HY_EUNSUPPORTED_TYPE; }
    if (m < 0) { set_error("%s: %d rows", what, m); return HY_EINVAL; }
    if (n <= 0 || k <= 0 || n > HY_MM_MAX || k > HY_MM_MAX || m > HY_MM_MAX) { set_error("%s: m %d, n %d, k %d (1 .. 2^30)", what, m, n, k); return HY_EBAD_SHAPE; }
    return HY_OK;
}
static int check_out_type(const char *what, int type, int out_type) {
    if (out_type != HY_F32 && out_type != type) { set_error("%s: output type %d (HY_F32 or the operands' type)", what, out_type); return HY_EUNSUPPORTED_TYPE; }
    return HY_OK;
}
// eight neighbouring values at columns that are multiples of 8 start on 16 bytes
static bool vec16(const void *p, int64_t ld, int bytes) { return !p || (ld % (16 / bytes) == 0 && !misaligned(p, 16)); }

#define HY_TRY(e) do { const int rc_ = (e); if (rc_ != HY_OK) return rc_; } while (0)

static MMArgs args() { MMArgs a{}; a.kq = a.kp = divisor(1); return a; }

// ------------------------------------------------------------------ experts

// the 16-bit layer descriptor: matrices [n_local][rows][cols], contiguous
static int check_dev16(const char *what, const hy_moe_dev *m, bool gate, bool down) {
    if (!m) { set_error("%s: null hy_moe_dev", what); return HY_EINVAL; }
    if (!m->slot || m->n_expert <= 0) { set_error("%s: slot table missing", what); return HY_EINVAL; }
    if (m->n_local <= 0 || m->n_local > 65535) { set_error("%s: n_local %d (1 .. 65535)", what, m->n_local); return HY_EINVAL; }
    if (m->ff <= 0 || m->n <= 0 || m->ff > HY_MM_MAX || m->n > HY_MM_MAX) { set_error("%s: ff %d, n %d", what, m->ff, m->n); return HY_EBAD_SHAPE; }
    const size_t bytes = 2 * (size_t) m->ff * (size_t) m->n;
    if (gate) {
        if (!type16(m->tg)) { set_error("%s: gate/up type %d (HY_F16 or HY_BF16)", what, m->tg); return HY_EUNSUPPORTED_TYPE; }
        if (!m->gate || !m->up) { set_error("%s: null gate/up", what); return HY_EINVAL; }
        if (m->gate_bytes != bytes) { set_error("%s: gate_bytes %zu != 2 ff n", what, m->gate_bytes); return HY_EBAD_SHAPE; }
        if (misaligned(m->gate, 2) || misaligned(m->up, 2)) { set_error("%s: gate/up must be 2-byte aligned", what); return HY_EBAD_SHAPE; }
    }
    if (down) {
        if (!type16(m->td)) { set_error("%s: down type %d (HY_F16 or HY_BF16)", what, m->td); return HY_EUNSUPPORTED_TYPE; }
        if (!m->down) { set_error("%s: null down", what); return HY_EINVAL; }
        if (m->down_bytes != bytes) { set_error("%s: down_bytes %zu != 2 ff n", what, m->down_bytes); return HY_EBAD_SHAPE; }
        if (misaligned(m->down, 2)) { set_error("%s: down must be 2-byte aligned", what); return HY_EBAD_SHAPE; }
    }
    return HY_OK;
}
static int check_k(const char *what, int k) {
    if (k < 1 || k > 64) { set_error("%s: k = %d pairs a row (1 .. 64)", what, k); return HY_EBAD_SHAPE; }
    return HY_OK;
}
// the pairs' grouping: order, order_n and egrp of hy_moe_order (without pairs nothing reads it: empty arrays have no address)
static int check_groups(const char *what, int n_pairs, const int32_t *order, const int32_t *order_n, const int32_t *egrp, int max_active) {
    if (n_pairs < 0) { set_error("%s: %d pairs", what, n_pairs); return HY_EINVAL; }
    if (n_pairs > HY_MM_MAX) { set_error("%s: %d pairs (up to 2^30)", what, n_pairs); return HY_EBAD_SHAPE; }
    if (n_pairs == 0) return HY_OK;
    if (!order || !order_n || !egrp) { set_error("%s: order, order_n and egrp are needed", what); return HY_EINVAL; }
    if (misaligned(order, 4) || misaligned(order_n, 4) || misaligned(egrp, 4)) { set_error("%s: order, order_n and egrp must be 4-byte aligned", what); return HY_EBAD_SHAPE; }
    if (max_active < 1 || max_active > 1024) { set_error("%s: max_active %d (1 .. 1024)", what, max_active); return HY_EBAD_SHAPE; }
    return HY_OK;
}
// by ids (order null) or grouped
static int check_pairs(const char *what, int n_pairs, const int32_t *ids, const int32_t *order, const int32_t *order_n, const int32_t *egrp,
                       int max_active) {
    if (order) return check_groups(what, n_pairs, order, order_n, egrp, max_active);
    if (n_pairs < 0) { set_error("%s: %d pairs", what, n_pairs); return HY_EINVAL; }
    if (n_pairs == 0) return HY_OK;
    if (!ids) { set_error("%s: ids or order is needed", what); return HY_EINVAL; }
    if (misaligned(ids, 4)) { set_error("%s: ids must be 4-byte aligned", what); return HY_EBAD_SHAPE; }
    if (n_pairs > 65535) { set_error("%s: %d pairs by ids (up to 65535: group them with hy_moe_order)", what, n_pairs); return HY_EBAD_SHAPE; }
    return HY_OK;
}
static MMArgs moe_args(const hy_moe_dev *m, int n_pairs, const int32_t *ids, const int32_t *order, const int32_t *order_n, const int32_t *egrp,
                       int max_active) {
    MMArgs a = args();
    a.slot = m->slot;
    a.n_local = m->n_local;
    a.n_expert = m->n_expert;
    a.n_pairs = n_pairs;
    a.pstride = (int64_t) m->ff * m->n;
    if (n_pairs == 0) return a;   // (gradients of no pairs: zeros)
    if (order) { a.order = order; a.order_n = order_n; a.egrp = egrp; a.max_active = max_active; }
    else a.ids = ids;
    return a;
}

} // namespace hy

using namespace hy;

extern "C" {

int hy_linear(int type, const void *W, int64_t ldw, int n, int k, const void *x, int64_t ldx, int m, const float *bias, int act,
              const void *resid, int64_t ldr, void *z, int64_t ldz, void *out, int out_type, int64_t ldo, hipStream_t s) {
    const char *what = "hy_linear";
    HY_TRY(check_sizes(what, type, m, n, k));
    HY_TRY(check_out_type(what, type, out_type));
    if (act < HY_ACT_NONE || act > HY_ACT_GELU_TANH) { set_error("%s: activation %d", what, act); return HY_EINVAL; }
    const int ob = out_type == HY_F32 ? 4 : 2;
    HY_TRY(check_mat(what, "W", W, ldw, n, k, 2, false));
    HY_TRY(check_mat(what, "x", x, ldx, m, k, 2, false));
    HY_TRY(check_mat(what, "out", out, ldo, m, n, ob, true));
    if (resid) HY_TRY(check_mat(what, "resid", resid, ldr, m, n, ob, false));
    if (z) HY_TRY(check_mat(what, "z", z, ldz, m, n, 2, true));
    if (bias && misaligned(bias, 4)) { set_error("%s: bias must be 4-byte aligned", what); return HY_EBAD_SHAPE; }
    if (m == 0) return HY_OK;
    MMArgs a = args();
    a.P = W; a.ldp = ldw; a.Q = x; a.ldq = ldx; a.R = m; a.N = n; a.K = k;
    a.bias = bias; a.act = act; a.resid = resid; a.ldr = ldr; a.z = z; a.ldz = ldz; a.out = out; a.ldo = ldo;
    a.out_f32 = out_type == HY_F32;
    a.bias16 = !misaligned(bias, 16);
    a.vec = vec16(out, ldo, ob) && vec16(resid, ldr, ob) && vec16(z, ldz, 2);
    return few_rows(a) ? launch_few(type, a, s, what) : m <= 4 ? launch_mv(type, false, a, s, what) : launch_mm(NT, type, false, a, s, what);
}

int hy_linear_glu(int type, const void *Wg, const void *Wu, int64_t ldw, int n, int k, const void *x, int64_t ldx, int m, float clamp,
                  void *g, void *u, void *h, int64_t ldh, hipStream_t s) {
    const char *what = "hy_linear_glu";
    HY_TRY(check_sizes(what, type, m, n, k));
    HY_TRY(check_mat(what, "Wg", Wg, ldw, n, k, 2, false));
    HY_TRY(check_mat(what, "Wu", Wu, ldw, n, k, 2, false));
    HY_TRY(check_mat(what, "x", x, ldx, m, k, 2, false));
    HY_TRY(check_mat(what, "h", h, ldh, m, n, 2, true));
    if (!g != !u) { set_error("%s: g and u go together", what); return HY_EINVAL; }
    if (g) { HY_TRY(check_mat(what, "g", g, ldh, m, n, 2, true)); HY_TRY(check_mat(what, "u", u, ldh, m, n, 2, true)); }
    if (m == 0) return HY_OK;
    MMArgs a = args();
    a.P = Wg; a.P2 = Wu; a.ldp = ldw; a.Q = x; a.ldq = ldx; a.R = m; a.N = n; a.K = k;
    a.g = g; a.u = u; a.out = h; a.ldo = ldh; a.clamp = clamp;
    a.vec = vec16(h, ldh, 2) && vec16(g, ldh, 2) && vec16(u, ldh, 2);
    return m <= 4 ? launch_mv(type, true, a, s, what) : launch_mm(NT, type, true, a, s, what);
}

int hy_act_bwd(int type, int act, const void *z, int64_t ldz, const void *dy, int64_t lddy, int m, int n, void *dz, int64_t lddz,
               hipStream_t s) {
    const char *what = "hy_act_bwd";
    HY_TRY(check_sizes(what, type, m, n, 1));
    if (act < HY_ACT_NONE || act > HY_ACT_GELU_TANH) { set_error("%s: activation %d", what, act); return HY_EINVAL; }
    HY_TRY(check_mat(what, "z", z, ldz, m, n, 2, false));
    HY_TRY(check_mat(what, "dy", dy, lddy, m, n, 2, false));
    HY_TRY(check_mat(what, "dz", dz, lddz, m, n, 2, true));
    return m == 0 ? HY_OK : launch_act_bwd(type, act, z, ldz, dy, lddy, m, n, dz, lddz, s);
}

int hy_linear_dx(int type, const void *W, int64_t ldw, int n, int k, const void *dz, int64_t lddz, int m, const void *resid, int64_t ldr,
                 void *dx, int out_type, int64_t lddx, hipStream_t s) {
    const char *what = "hy_linear_dx";
    HY_TRY(check_sizes(what, type, m, n, k));
    HY_TRY(check_out_type(what, type, out_type));
    const int ob = out_type == HY_F32 ? 4 : 2;
    HY_TRY(check_mat(what, "W", W, ldw, n, k, 2, false));
    HY_TRY(check_mat(what, "dz", dz, lddz, m, n, 2, false));
    HY_TRY(check_mat(what, "dx", dx, lddx, m, k, ob, true));
    if (resid) HY_TRY(check_mat(what, "resid", resid, ldr, m, k, ob, false));
    if (m == 0) return HY_OK;
    MMArgs a = args();
    a.P = W; a.ldp = ldw; a.Q = dz; a.ldq = lddz; a.R = m; a.N = k; a.K = n;
    a.resid = resid; a.ldr = ldr; a.out = dx; a.ldo = lddx; a.out_f32 = out_type == HY_F32;
    a.vec = vec16(dx, lddx, ob) && vec16(resid, ldr, ob);
    return launch_mm(NN, type, false, a, s, what);
}

size_t hy_linear_dw_ws_bytes(int m, int n, int k) {
    if (m <= 0 || n <= 0 || k <= 0 || m > HY_MM_MAX || n > HY_MM_MAX || k > HY_MM_MAX) return 0;
    const Parts p = dw_parts(m, n, k);
    return p.n > 1 ? (size_t) p.n * ((size_t) n * k + n) * 4 : 0;
}
int hy_linear_dw(int type, const void *dz, int64_t lddz, const void *x, int64_t ldx, int m, int n, int k, void *dW, int out_type,
                 int64_t lddw, float *db, int accumulate, void *ws, size_t ws_bytes, hipStream_t s) {
    const char *what = "hy_linear_dw";
    HY_TRY(check_sizes(what, type, m, n, k));
    HY_TRY(check_out_type(what, type, out_type));
    const int ob = out_type == HY_F32 ? 4 : 2;
    HY_TRY(check_mat(what, "dz", dz, lddz, m, n, 2, false));
    HY_TRY(check_mat(what, "x", x, ldx, m, k, 2, false));
    HY_TRY(check_mat(what, "dW", dW, lddw, n, k, ob, true));
    if (db && misaligned(db, 4)) { set_error("%s: db must be 4-byte aligned", what); return HY_EBAD_SHAPE; }
    const size_t need = hy_linear_dw_ws_bytes(m, n, k);
    if (need && (!ws || ws_bytes < need)) { set_error("%s: workspace of %zu bytes, %zu needed", what, ws ? ws_bytes : (size_t) 0, need); return HY_EINVAL; }
    if (need && misaligned(ws, 16)) { set_error("%s: the workspace must be 16-byte aligned", what); return HY_EBAD_SHAPE; }
    MMArgs a = args();
    a.P = x; a.ldp = ldx; a.Q = dz; a.ldq = lddz; a.R = n; a.N = k; a.K = m;
    a.out = dW; a.ldo = lddw; a.out_f32 = out_type == HY_F32; a.db = db; a.accumulate = accumulate != 0;
    a.vec = vec16(dW, lddw, ob);
    if (need) {
        const Parts p = dw_parts(m, n, k);
        a.part = (float *) ws; a.parts = p.n; a.part_len = p.len;
    }
    return launch_mm(TN, type, false, a, s, what);
}

int hy_moe16_gate_up(const hy_moe_dev *m, const void *x, int64_t ldx, int k, const int32_t *ids, int n_pairs, const int32_t *order,
                     const int32_t *order_n, const int32_t *egrp, int max_active, void *g, void *u, void *h, hipStream_t s) {
    const char *what = "hy_moe16_gate_up";
    HY_TRY(check_dev16(what, m, true, false));
    HY_TRY(check_k(what, k));
    HY_TRY(check_pairs(what, n_pairs, ids, order, order_n, egrp, max_active));
    HY_TRY(check_mat(what, "x", x, ldx, n_pairs, m->n, 2, false));
    HY_TRY(check_mat(what, "h", h, m->ff, n_pairs, m->ff, 2, true));
    if (!g != !u) { set_error("%s: g and u go together", what); return HY_EINVAL; }
    if (g && (misaligned(g, 2) || misaligned(u, 2))) { set_error("%s: g and u must be 2-byte aligned", what); return HY_EBAD_SHAPE; }
    if (n_pairs == 0) return HY_OK;
    MMArgs a = moe_args(m, n_pairs, ids, order, order_n, egrp, max_active);
    a.P = m->gate; a.P2 = m->up; a.ldp = m->n; a.Q = x; a.ldq = ldx; a.kq = divisor((uint32_t) k); a.N = m->ff; a.K = m->n; a.R = 1;
    a.g = g; a.u = u; a.out = h; a.ldo = m->ff; a.clamp = m->clamp;
    a.vec = vec16(h, m->ff, 2) && vec16(g, m->ff, 2) && vec16(u, m->ff, 2);
    return order ? launch_mm(NT, m->tg, true, a, s, what) : launch_mv(m->tg, true, a, s, what);
}

int hy_moe16_down(const hy_moe_dev *m, const void *h, const int32_t *ids, int n_pairs, const int32_t *order, const int32_t *order_n,
                  const int32_t *egrp, int max_active, const float *wts, void *y, int out_type, hipStream_t s) {
    const char *what = "hy_moe16_down";
    HY_TRY(check_dev16(what, m, false, true));
    HY_TRY(check_out_type(what, m->td, out_type));
    HY_TRY(check_pairs(what, n_pairs, ids, order, order_n, egrp, max_active));
    const int ob = out_type == HY_F32 ? 4 : 2;
    HY_TRY(check_mat(what, "h", h, m->ff, n_pairs, m->ff, 2, false));
    HY_TRY(check_mat(what, "y", y, m->n, n_pairs, m->n, ob, true));
    if (wts && misaligned(wts, 4)) { set_error("%s: wts must be 4-byte aligned", what); return HY_EBAD_SHAPE; }
    if (n_pairs == 0) return HY_OK;
    MMArgs a = moe_args(m, n_pairs, ids, order, order_n, egrp, max_active);
    a.P = m->down; a.ldp = m->ff; a.Q = h; a.ldq = m->ff; a.N = m->n; a.K = m->ff; a.R = 1;
    a.wts = wts; a.out = y; a.ldo = m->n; a.out_f32 = out_type == HY_F32;
    a.vec = vec16(y, m->n, ob);
    return order ? launch_mm(NT, m->td, false, a, s, what) : launch_mv(m->td, false, a, s, what);
}

int hy_moe16_reduce(const hy_moe_dev *m, const float *shexp, const float *sg, const float *y, int k, float *out, int nt, const int32_t *ids,
                    hipStream_t s) {
    const char *what = "hy_moe16_reduce";
    HY_TRY(check_dev16(what, m, false, false));
    HY_TRY(check_k(what, k));
    if (nt < 0 || nt > HY_MM_MAX / k) { set_error("%s: %d rows of %d pairs (up to 2^30 pairs)", what, nt, k); return nt < 0 ? HY_EINVAL : HY_EBAD_SHAPE; }
    if (nt == 0) return HY_OK;
    if (!y || !out || !ids) { set_error("%s: null y, out or ids", what); return HY_EINVAL; }
    if (misaligned(shexp, 4) || misaligned(sg, 4) || misaligned(y, 4) || misaligned(out, 4) || misaligned(ids, 4)) { set_error("%s: arguments must be 4-byte aligned", what); return HY_EBAD_SHAPE; }
    return launch_reduce_local(*m, shexp, sg, y, k, out, nt, ids, s);
}

int hy_moe16_down_dx(const hy_moe_dev *m, const void *dy, int64_t lddy, int k, int n_pairs, const int32_t *order, const int32_t *order_n,
                     const int32_t *egrp, int max_active, void *dh, int out_type, hipStream_t s) {
    const char *what = "hy_moe16_down_dx";
    HY_TRY(check_dev16(what, m, false, true));
    HY_TRY(check_out_type(what, m->td, out_type));
    HY_TRY(check_k(what, k));
    HY_TRY(check_groups(what, n_pairs, order, order_n, egrp, max_active));
    const int ob = out_type == HY_F32 ? 4 : 2;
    HY_TRY(check_mat(what, "dy", dy, lddy, n_pairs, m->n, 2, false));
    HY_TRY(check_mat(what, "dh", dh, m->ff, n_pairs, m->ff, ob, true));
    if (n_pairs == 0) return HY_OK;
    MMArgs a = moe_args(m, n_pairs, nullptr, order, order_n, egrp, max_active);
    a.P = m->down; a.ldp = m->ff; a.Q = dy; a.ldq = lddy; a.kq = divisor((uint32_t) k); a.N = m->ff; a.K = m->n;
    a.out = dh; a.ldo = m->ff; a.out_f32 = out_type == HY_F32;
    a.vec = vec16(dh, m->ff, ob);
    return launch_mm(NN, m->td, false, a, s, what);
}

int hy_moe16_gate_up_dx(const hy_moe_dev *m, const void *dg, const void *du, int n_pairs, const int32_t *order, const int32_t *order_n,
                        const int32_t *egrp, int max_active, void *dx, int out_type, hipStream_t s) {
    const char *what = "hy_moe16_gate_up_dx";
    HY_TRY(check_dev16(what, m, true, false));
    HY_TRY(check_out_type(what, m->tg, out_type));
    HY_TRY(check_groups(what, n_pairs, order, order_n, egrp, max_active));
    const int ob = out_type == HY_F32 ? 4 : 2;
    HY_TRY(check_mat(what, "dg", dg, m->ff, n_pairs, m->ff, 2, false));
    HY_TRY(check_mat(what, "du", du, m->ff, n_pairs, m->ff, 2, false));
    HY_TRY(check_mat(what, "dx", dx, m->n, n_pairs, m->n, ob, true));
    if (n_pairs == 0) return HY_OK;
    MMArgs a = moe_args(m, n_pairs, nullptr, order, order_n, egrp, max_active);
    a.P = m->gate; a.P2 = m->up; a.ldp = m->n; a.Q = dg; a.Q2 = du; a.ldq = m->ff; a.N = m->n; a.K = m->ff;
    a.out = dx; a.ldo = m->n; a.out_f32 = out_type == HY_F32;
    a.vec = vec16(dx, m->n, ob);
    return launch_mm(NN, m->tg, false, a, s, what);
}

int hy_moe16_dw(const hy_moe_dev *m, int type, const void *a_, int64_t lda, int ka, int rows, const void *b, int64_t ldb, int kb, int cols,
                int n_pairs, const int32_t *order, const int32_t *order_n, const int32_t *egrp, int max_active, void *dW, int out_type,
                int accumulate, hipStream_t s) {
    const char *what = "hy_moe16_dw";
    HY_TRY(check_dev16(what, m, false, false));
    HY_TRY(check_sizes(what, type, n_pairs, rows, cols));
    HY_TRY(check_out_type(what, type, out_type));
    HY_TRY(check_k(what, ka));
    HY_TRY(check_k(what, kb));
    HY_TRY(check_groups(what, n_pairs, order, order_n, egrp, max_active));
    const int ob = out_type == HY_F32 ? 4 : 2;
    HY_TRY(check_mat(what, "a", a_, lda, n_pairs, rows, 2, false));
    HY_TRY(check_mat(what, "b", b, ldb, n_pairs, cols, 2, false));
    HY_TRY(check_mat(what, "dW", dW, cols, rows, cols, ob, true));
    MMArgs a = moe_args(m, n_pairs, nullptr, order, order_n, egrp, max_active);
    a.P = b; a.ldp = ldb; a.kp = divisor((uint32_t) kb); a.Q = a_; a.ldq = lda; a.kq = divisor((uint32_t) ka); a.R = rows; a.N = cols;
    a.out = dW; a.ldo = cols; a.ostride = (int64_t) rows * cols; a.out_f32 = out_type == HY_F32; a.accumulate = accumulate != 0;
    a.vec = vec16(dW, cols, ob);
    return launch_mm(TN, type, false, a, s, what);
}

int hy_swiglu_bwd(int type, const void *g, const void *u, const void *dh, const float *wts, int n_pairs, int ff, float clamp,
                  const int32_t *order, const int32_t *order_n, void *dg, void *du, void *hw, float *dwts, hipStream_t s) {
    const char *what = "hy_swiglu_bwd";
    HY_TRY(check_sizes(what, type, n_pairs, ff, 1));
    HY_TRY(check_mat(what, "g", g, ff, n_pairs, ff, 2, false));
    HY_TRY(check_mat(what, "u", u, ff, n_pairs, ff, 2, false));
    HY_TRY(check_mat(what, "dh", dh, ff, n_pairs, ff, 2, false));
    HY_TRY(check_mat(what, "dg", dg, ff, n_pairs, ff, 2, true));
    HY_TRY(check_mat(what, "du", du, ff, n_pairs, ff, 2, true));
    if (hw) HY_TRY(check_mat(what, "hw", hw, ff, n_pairs, ff, 2, true));
    if (!order != !order_n) { set_error("%s: order and order_n go together", what); return HY_EINVAL; }
    if (misaligned(wts, 4) || misaligned(dwts, 4) || misaligned(order, 4) || misaligned(order_n, 4)) { set_error("%s: wts, dwts, order and order_n must be 4-byte aligned", what); return HY_EBAD_SHAPE; }
    return n_pairs == 0 ? HY_OK : launch_swiglu_bwd(type, g, u, dh, wts, n_pairs, ff, clamp, order, order_n, dg, du, hw, dwts, s);
}

int hy_rows16(int type, const float *x, int64_t xs, int n, int nt, void *out, int64_t ldo, hipStream_t s) {
    const char *what = "hy_rows16";
    HY_TRY(check_sizes(what, type, nt, n, 1));
    HY_TRY(check_mat(what, "x", x, xs, nt, n, 4, false));
    HY_TRY(check_mat(what, "out", out, ldo, nt, n, 2, true));
    return nt == 0 ? HY_OK : launch_rows16(type, x, xs, n, nt, out, ldo, s);
}

} // extern "C"
