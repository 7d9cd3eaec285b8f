"""16-bit matrix products against 64-bit formulas.

Products are mostly tested on small integers: every product and partial sum is then an integer below 2^24, exact in any order
of fp32 sums, so a float32 output equals the formula's bit for bit and a 16-bit output is its nearest value.  Where an
activation follows, the bound counts: (K + 4) 2^-23 sum |w x| for the sum (one unit in the last place of the largest partial
sum a term, whether sums round or truncate), times the activation's steepest slope (at most 1.13), a few 2^-24 of evaluation,
and half a step of the output's type."""
import math

import numpy as np
import pytest
import torch

from hyper_amd import mm16, moe
from tests.helpers import gen

pytestmark = pytest.mark.gpu

TYPES = [torch.bfloat16, torch.float16]
NAN = float("nan")


def ints(g, *shape, lo=-3, hi=3):
    return torch.randint(lo, hi + 1, shape, generator=g).double()


def put(t, dtype, dev, pad=0, offset=0):
    """t on the device as dtype; pad / offset: a view of a wider matrix filled with NaN, `offset` elements off its start"""
    if not pad and not offset:
        return t.to(dtype).to(dev)
    flat = torch.full((t.shape[0] * (t.shape[1] + pad) + offset,), NAN, dtype=dtype, device=dev)
    v = flat[offset:].view(t.shape[0], t.shape[1] + pad)[:, :t.shape[1]]
    v.copy_(t.to(dtype))
    return v


def empty(m, n, dtype, dev, pad=0, offset=0):
    """an output of m x n inside a buffer of sentinels; returns (view, check of what lies around it)"""
    flat = torch.full((m * (n + pad) + offset + 64,), 77.0, dtype=dtype, device=dev)
    v = flat[offset:offset + m * (n + pad)].view(m, n + pad)[:, :n]

    def untouched():
        rest = flat.clone()
        rest[offset:offset + m * (n + pad)].view(m, n + pad)[:, :n] = 77.0
        assert (rest == 77.0).all(), "values around the output were written"
    return v, untouched


def same(got, want, what=""):
    """bit for bit the nearest value of got's type"""
    w = want.to(torch.float32).to(got.dtype).cpu()
    g = got.cpu()
    assert g.shape == w.shape, (what, g.shape, w.shape)
    bad = ~((g == w) | (g.isnan() & w.isnan()))
    assert not bad.any(), f"{what}: {int(bad.sum())} of {bad.numel()} differ, first at {bad.nonzero()[0].tolist()}: {g[bad][0]} for {w[bad][0]}"


def act64(name, z):
    if name == "relu":
        return z.clamp_min(0)
    if name == "silu":
        return z * torch.sigmoid(z)
    if name == "gelu":
        return 0.5 * z * torch.erfc(-z / math.sqrt(2))
    if name == "gelu_tanh":
        return 0.5 * z * (1 + torch.tanh(math.sqrt(2 / math.pi) * (z + 0.044715 * z ** 3)))
    return z


def half(dtype, v):
    """half a step of dtype at |v|, and of its smallest values"""
    tiny = {torch.bfloat16: 2.0 ** -134, torch.float16: 2.0 ** -25, torch.float32: 2.0 ** -150}[dtype]
    return v.abs() * torch.finfo(dtype).eps / 2 + tiny


def within(got, want, err, what=""):
    """|got - want| <= err (before rounding) plus got's own rounding"""
    bound = err + half(got.dtype, want.abs() + err)
    off = (got.double().cpu() - want).abs()
    # a value at or beyond the largest finite one plus half its step (fp16: 65504 + 16) rounds to infinity of its sign
    top = torch.finfo(got.dtype).max * (1 + torch.finfo(got.dtype).eps / 4)
    bad = ~(off <= bound) & ~((got.double().cpu() == want.sign() * float("inf")) & (want.abs() + err >= top))
    assert not bad.any(), f"{what}: {int(bad.sum())} of {bad.numel()} off, first at {bad.nonzero()[0].tolist()}: {off[bad][0]:.3g} > {bound[bad][0]:.3g}"


def glu_err(want, u):
    """evaluation of silu(g) u for exact g and u: a few 2^-24, and below g = -87.33, where 1 / (1 + exp(-g)) leaves the normal
    numbers and is 0, the value itself: |g| exp(g) < 87.34 exp(-87.33) < 1.04e-36 there, times |u|"""
    return 16 * 2.0 ** -24 * want.abs() + 1.04e-36 * u.abs()


# (rows, outputs, inputs): one row to many, sizes around the tiles, odd ones, rows that are and are not multiples of 16 bytes
SIZES = [(1, 1, 1), (1, 64, 64), (1, 2048, 2048), (2, 100, 72), (3, 37, 515), (4, 129, 256), (5, 16, 8), (7, 40, 33), (15, 264, 136),
         (16, 128, 64), (17, 130, 200), (33, 72, 1024), (63, 65, 127), (64, 256, 128), (100, 260, 72), (129, 129, 129), (200, 520, 328),
         (256, 256, 256), (300, 1000, 264), (513, 384, 1032), (1025, 264, 520)]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("m,n,k", SIZES)
def test_linear(cuda, dtype, m, n, k):
    g = gen(m * 7919 + n * 31 + k)
    W, x = ints(g, n, k), ints(g, m, k)
    bias, resid = ints(g, n), ints(g, m, n)
    z = x @ W.t()
    Wd, xd = put(W, dtype, cuda), put(x, dtype, cuda)
    for out_t in (dtype, torch.float32):
        out, ok = empty(m, n, out_t, cuda)
        mm16.linear(Wd, xd, out)
        same(out, z, f"plain {out_t}")
        zt, okz = empty(m, n, dtype, cuda)
        mm16.linear(Wd, xd, out, bias=bias.float().to(cuda), act="relu", resid=resid.to(out_t).to(cuda), z=zt)
        same(out, (z + bias).clamp_min(0) + resid, f"epilogue {out_t}")
        same(zt, z + bias, "z")
        res = resid.to(out_t).to(cuda)
        mm16.linear(Wd, xd, res, resid=res)                   # in place
        same(res, z + resid, f"residual in place {out_t}")
        ok(), okz()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("m,n,k", [(1, 64, 64), (3, 37, 515), (5, 24, 40), (40, 100, 72), (130, 264, 136), (300, 1000, 264)])
@pytest.mark.parametrize("pad,offset", [(8, 0), (5, 0), (8, 8), (0, 1), (16, 4), (3, 3)])
def test_linear_strides(cuda, dtype, m, n, k, pad, offset):
    """rows apart in wider matrices (NaN between them), starts off 16 bytes: nothing around a row is read into it or written"""
    g = gen(m + 13 * n + 7 * k + pad)
    W, x, resid = ints(g, n, k), ints(g, m, k), ints(g, m, n)
    Wd, xd = put(W, dtype, cuda, pad, offset), put(x, dtype, cuda, pad, offset)
    for out_t in (dtype, torch.float32):
        out, ok = empty(m, n, out_t, cuda, pad, offset)
        z, okz = empty(m, n, dtype, cuda, pad, offset)
        mm16.linear(Wd, xd, out, resid=put(resid, out_t, cuda, pad, offset), z=z)
        same(out, x @ W.t() + resid, "out")
        same(z, x @ W.t(), "z")
        ok(), okz()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("act", list(mm16.ACTS))
@pytest.mark.parametrize("m,n,k", [(1, 200, 512), (3, 96, 100), (40, 130, 256), (300, 264, 1024)])
def test_linear_activations(cuda, dtype, act, m, n, k):
    g = gen(m + n + k)
    W, x = (torch.randn(n, k, generator=g) * 2 / math.sqrt(k)).to(dtype), torch.randn(m, k, generator=g).to(dtype)
    bias = torch.randn(n, generator=g)
    z = x.double() @ W.double().t() + bias.double()
    mag = x.double().abs() @ W.double().abs().t() + bias.double().abs()
    err = 1.13 * (k + 4) * 2.0 ** -23 * mag + 16 * 2.0 ** -24 * (z.abs() + 1)
    for out_t in (dtype, torch.float32):
        out = torch.empty(m, n, dtype=out_t, device=cuda)
        mm16.linear(W.to(cuda), x.to(cuda), out, bias=bias.to(cuda), act=act)
        within(out, act64(act, z), err, f"{act} {out_t}")


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("m,n,k", [(1, 64, 64), (2, 33, 40), (6, 17, 24), (40, 100, 72), (130, 264, 136), (300, 520, 264)])
@pytest.mark.parametrize("clamp", [0.0, 7.0])
def test_linear_glu(cuda, dtype, m, n, k, clamp):
    g = gen(m + n + k)
    Wg, Wu, x = ints(g, n, k), ints(g, n, k), ints(g, m, k)
    G, U = x @ Wg.t(), x @ Wu.t()
    h, ok = empty(m, n, dtype, cuda)
    gd, okg = empty(m, n, dtype, cuda)
    ud, oku = empty(m, n, dtype, cuda)
    a = put(Wg, dtype, cuda), put(Wu, dtype, cuda), put(x, dtype, cuda)
    mm16.linear_glu(*a, h, clamp=clamp, g=gd, u=ud)
    same(gd, G, "g"), same(ud, U, "u")
    if clamp:
        G, U = G.clamp_max(clamp), U.clamp(-clamp, clamp)
    want = G * torch.sigmoid(G) * U                             # g and u are exact: only their product's evaluation is off
    within(h, want, glu_err(want, U), "h")
    h2 = torch.empty_like(h.contiguous())
    mm16.linear_glu(*a, h2, clamp=clamp)
    assert torch.equal(h2, h)
    ok(), okg(), oku()


GRAD_SIZES = [(0, 24, 16), (1, 8, 8), (1, 40, 33), (3, 130, 72), (16, 64, 64), (33, 129, 65), (64, 128, 256), (100, 264, 136), (257, 65, 520),
              (300, 512, 264), (1000, 48, 40), (513, 260, 264), (5000, 64, 72), (4097, 136, 520)]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("m,n,k", GRAD_SIZES)
@pytest.mark.parametrize("pad,offset", [(0, 0), (8, 8), (3, 1)])
def test_linear_gradients(cuda, dtype, m, n, k, pad, offset):
    g = gen(m * 17 + n + k)
    W, x, dz, resid = ints(g, n, k), ints(g, m, k), ints(g, m, n), ints(g, m, k)
    Wd, xd, dzd = (put(t, dtype, cuda, pad, offset) for t in (W, x, dz))
    for out_t in (dtype, torch.float32):
        dx, ok = empty(m, k, out_t, cuda, pad, offset)
        mm16.linear_dx(Wd, dzd, dx)
        same(dx, dz @ W, "dx")
        mm16.linear_dx(Wd, dzd, dx, resid=put(resid, out_t, cuda, pad, offset))
        same(dx, dz @ W + resid, "dx + resid")
        ok()
        dW, ok = empty(n, k, out_t, cuda, pad, offset)
        db = torch.full((n + 3,), 77.0, device=cuda)
        ws = torch.empty(mm16.linear_dw_ws_bytes(m, n, k), dtype=torch.uint8, device=cuda)
        mm16.linear_dw(dzd, xd, dW, db=db, ws=ws)
        same(dW, dz.t() @ x, "dW")
        same(db[:n], dz.sum(0), "db")
        assert (db[n:] == 77.0).all()
        dW2, _ = empty(n, k, out_t, cuda, pad, offset)
        mm16.linear_dw(dzd, xd, dW2, ws=ws)
        same(dW2, dz.t() @ x, "dW without db")
        dW.fill_(5.0)
        db.fill_(2.0)
        mm16.linear_dw(dzd, xd, dW, db=db, accumulate=True, ws=ws)
        same(dW, dz.t() @ x + 5, "dW accumulated")
        same(db[:n], dz.sum(0) + 2, "db accumulated")
        ok()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("act", list(mm16.ACTS))
@pytest.mark.parametrize("m,n,pad", [(1, 8, 0), (3, 37, 0), (40, 96, 8), (5, 64, 3)])
def test_act_bwd(cuda, dtype, act, m, n, pad):
    """against the 64-bit derivative, taken by differences of the 64-bit formula with step 2^-17 (error of a central
    difference: h^2 / 6 |act'''| < 1e-10; relu away from 0)"""
    g = gen(n)
    z, dy = (torch.randn(m, n, generator=g) * 3).to(dtype), torch.randn(m, n, generator=g).to(dtype)
    z.view(-1)[0] = 1.0
    zd, step = z.double(), 2.0 ** -17
    z = torch.where(zd.abs() < 1e-3, torch.ones_like(z), z)
    zd = z.double()
    d = (act64(act, zd + step) - act64(act, zd - step)) / (2 * step)
    out, ok = empty(m, n, dtype, cuda, pad)
    mm16.act_bwd(act, put(z.float(), dtype, cuda, pad), put(dy.float(), dtype, cuda, pad), out)
    within(out, dy.double() * d, dy.double().abs() * (1e-8 + 32 * 2.0 ** -24 * (1 + zd.abs())), act)
    ok()
    both = dy.to(cuda)
    mm16.act_bwd(act, z.to(cuda), both, both)                  # in place
    assert torch.equal(both, out.contiguous())
    # both sides of zero, and values whose exponentials leave the range
    e = torch.tensor([[0.0, -0.0, 100.0, -100.0, 80.0, -80.0, 10.0, -10.0]], dtype=dtype, device=cuda)
    one = torch.ones_like(e)
    mm16.act_bwd(act, e, one, e)
    want = {"none": [1] * 8, "relu": [0, 0, 1, 0, 1, 0, 1, 0]}.get(act, [0.5, 0.5, 1, 0, 1, 0, None, None])
    for v, w in zip(e.cpu().view(-1).tolist(), want):
        assert w is None or abs(v - w) < 1e-6, (act, e)


# ------------------------------------------------------------------ experts

def route(g, T, E, k, kind):
    """ids [T k]: distinct experts a token; spread, all on the same k, or skewed with experts that get nothing"""
    if kind == "same":
        return torch.arange(k).repeat(T).to(torch.int32) + (E - k)
    p = torch.ones(E) if kind == "even" else 1.0 / torch.arange(1, E + 1).float() ** 2
    return torch.stack([torch.multinomial(p + 1e-9, k, generator=g) for _ in range(T)]).reshape(-1).to(torch.int32)


class Layer:
    """integer experts of the sizes, some absent (slot -1) when `missing`, and the grouping hy_moe_order makes"""

    def __init__(self, cuda, dtype, T, d, E, k, ff, kind="even", missing=False, clamp=0.0, seed=0, lo=-2, hi=2, offset=0):
        g = gen(1000 * T + d + E + ff + seed)
        self.ids = route(g, T, E, k, kind)
        slot = torch.arange(E, dtype=torch.int32)
        if missing:
            slot = torch.tensor([-1 if e % 3 == 1 else 0 for e in range(E)], dtype=torch.int32)
            slot[slot == 0] = torch.randperm(int((slot == 0).sum()), generator=g).to(torch.int32)
        self.slot, self.nl = slot, int((slot >= 0).sum())
        self.gate, self.up, self.down = ints(g, self.nl, ff, d, lo=lo, hi=hi), ints(g, self.nl, ff, d, lo=lo, hi=hi), ints(g, self.nl, d, ff, lo=lo, hi=hi)
        self.x, self.P, self.k, self.T, self.E, self.d, self.ff, self.g = ints(g, T, d), T * k, k, T, E, d, ff, g
        self.wts = 2.0 ** -torch.randint(0, 4, (self.P,), generator=g).double()
        on = lambda t: put(t.reshape(-1, t.shape[-1]), dtype, cuda, 0, offset).view(t.shape)  # noqa: E731
        self.dev = mm16.Moe16Dev(on(self.gate), on(self.up), on(self.down), slot.to(cuda), clamp)
        i32 = dict(dtype=torch.int32, device=cuda)
        self.ids_d = self.ids.to(cuda)
        self.order, self.order_n, self.egrp = torch.zeros(max(self.P, 1), **i32), torch.zeros(2, **i32), torch.zeros(3 * E, **i32)
        moe.moe_order(self.dev, self.ids_d, self.P, E, self.order, self.order_n, None, self.egrp)
        self.ma = max(1, min(E, self.P))
        self.grp = (self.order, self.order_n, self.egrp, self.ma)
        self.kw = dict(order=self.order, order_n=self.order_n, egrp=self.egrp, max_active=self.ma)
        self.local = slot[self.ids.long()] >= 0
        self.le = slot[self.ids.long()].long()
        self.tok = torch.arange(self.P) // k

    def fwd(self, W, rows):
        """rows[p] W[le[p]]^T, zeros for absent experts"""
        out = torch.zeros(self.P, W.shape[1], dtype=torch.float64)
        for e in range(self.nl):
            p = (self.local & (self.le == e)).nonzero().view(-1)
            out[p] = rows[p] @ W[e].t()
        return out

    def dw(self, a, b):
        out = torch.zeros(self.nl, a.shape[1], b.shape[1], dtype=torch.float64)
        for e in range(self.nl):
            p = (self.local & (self.le == e)).nonzero().view(-1)
            out[e] = a[p].t() @ b[p]
        return out


def same_rows(got, want, local, what):
    same(got[local.to(got.device)], want[local], what)
    assert (got[~local.to(got.device)] == 77.0).all(), f"{what}: rows of absent experts were written"


def marked(dev, dtype, *shape):
    return torch.full(shape, 77.0, dtype=dtype, device=dev)


# tokens, d, E, k, ff, routing
MOE = [(1, 64, 8, 2, 32, "even"), (1, 2048, 16, 8, 768, "even"), (2, 72, 5, 3, 40, "even"), (3, 33, 4, 1, 17, "even"), (9, 128, 16, 4, 96, "skew"),
       (37, 264, 20, 8, 136, "even"), (64, 256, 4, 2, 256, "same"), (100, 520, 64, 6, 72, "skew"), (150, 128, 3, 2, 264, "even"),
       (333, 136, 512, 10, 64, "even"), (300, 264, 6, 2, 520, "skew"), (700, 72, 2, 1, 512, "even")]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("T,d,E,k,ff,kind", MOE)
@pytest.mark.parametrize("missing", [False, True])
def test_expert_products(cuda, dtype, T, d, E, k, ff, kind, missing):
    L = Layer(cuda, dtype, T, d, E, k, ff, kind, missing)
    xp = L.x[L.tok]
    G, U = L.fwd(L.gate, xp), L.fwd(L.up, xp)
    xd, hrows = put(L.x, dtype, cuda, 8), ints(L.g, L.P, ff)
    hd = hrows.to(dtype).to(cuda)
    for how in ((L.kw, dict(ids=L.ids_d)) if T <= 9 else (L.kw,)):
        h, g, u = (marked(cuda, dtype, L.P, ff) for _ in range(3))
        mm16.moe16_gate_up(L.dev, xd, k, L.P, h, **how, g=g, u=u)
        same_rows(g, G, L.local, "g")
        same_rows(u, U, L.local, "u")
        want = G * torch.sigmoid(G) * U
        loc = L.local
        within(h[loc.to(cuda)], want[loc], glu_err(want[loc], U[loc]), "h")
        assert (h[~loc.to(cuda)] == 77.0).all()
        h2 = marked(cuda, dtype, L.P, ff)
        mm16.moe16_gate_up(L.dev, xd, k, L.P, h2, **how)
        assert torch.equal(h2, h)
        for out_t in (dtype, torch.float32):
            y = marked(cuda, out_t, L.P, d)
            mm16.moe16_down(L.dev, hd, L.P, y, wts=L.wts.float().to(cuda), **how)
            same_rows(y, L.fwd(L.down, hrows) * L.wts[:, None], L.local, f"y {out_t}")
            y = marked(cuda, out_t, L.P, d)
            mm16.moe16_down(L.dev, hd, L.P, y, **how)
            same_rows(y, L.fwd(L.down, hrows), L.local, f"y unweighted {out_t}")


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("T,d,E,k,ff,kind", MOE)
@pytest.mark.parametrize("missing", [False, True])
def test_expert_gradients(cuda, dtype, T, d, E, k, ff, kind, missing):
    L = Layer(cuda, dtype, T, d, E, k, ff, kind, missing, seed=1)
    dy, dg, du, hw = ints(L.g, T, d), ints(L.g, L.P, ff), ints(L.g, L.P, ff), ints(L.g, L.P, ff)
    on = lambda t: t.to(dtype).to(cuda)  # noqa: E731
    dyd, dgd, dud, hwd, xd = put(dy, dtype, cuda, 8), on(dg), on(du), on(hw), on(L.x)
    for out_t in (dtype, torch.float32):
        dh = marked(cuda, out_t, L.P, ff)
        mm16.moe16_down_dx(L.dev, dyd, k, L.P, *L.grp, dh)
        same_rows(dh, L.fwd(L.down.transpose(1, 2), dy[L.tok]), L.local, "dh")
        dx = marked(cuda, out_t, L.P, d)
        mm16.moe16_gate_up_dx(L.dev, dgd, dud, L.P, *L.grp, dx)
        same_rows(dx, L.fwd(L.gate.transpose(1, 2), dg) + L.fwd(L.up.transpose(1, 2), du), L.local, "dx")
        for name, a, ka, A, b, kb, B in (("gate", dgd, 1, dg, xd, k, L.x[L.tok]), ("down", dyd, k, dy[L.tok], hwd, 1, hw)):
            want = L.dw(A, B)
            dW = marked(cuda, out_t, L.nl, *want.shape[1:])
            mm16.moe16_dw(L.dev, a, ka, b, kb, L.P, *L.grp, dW)
            same(dW, want, f"dW {name} {out_t}")                 # zeros where an expert has no pairs
            dW.fill_(3.0)
            mm16.moe16_dw(L.dev, a, ka, b, kb, L.P, *L.grp, dW, accumulate=True)
            same(dW, want + 3, f"dW {name} accumulated {out_t}")


@pytest.mark.parametrize("dtype", TYPES)
def test_expert_no_pairs(cuda, dtype):
    """no tokens: nothing is written but the weights' gradients, which are zeros; every expert absent: no rows"""
    L = Layer(cuda, dtype, 4, 64, 8, 2, 32)
    h = marked(cuda, dtype, 8, 32)
    mm16.moe16_gate_up(L.dev, put(L.x, dtype, cuda), 2, 0, h, **L.kw)
    assert (h == 77.0).all()
    L.order_n.zero_()
    mm16.moe16_gate_up(L.dev, put(L.x, dtype, cuda), 2, 8, h, **L.kw)
    assert (h == 77.0).all()
    dW = marked(cuda, dtype, 8, 32, 64)
    mm16.moe16_dw(L.dev, h, 1, put(L.x, dtype, cuda), 2, 8, *L.grp, dW)
    assert (dW == 0).all()
    dW = marked(cuda, torch.float32, 8, 32, 64)
    mm16.moe16_dw(L.dev, h, 1, put(L.x, dtype, cuda), 2, 0, *L.grp, dW)
    assert (dW == 0).all()


def test_expert_bad_tables(cuda):
    """grouping tables that name no pair, expert or matrix are skipped: nothing outside the buffers is read or written"""
    L = Layer(cuda, torch.bfloat16, 6, 64, 8, 2, 32)
    x = put(L.x, torch.bfloat16, cuda)
    for spoil in ("expert", "start", "count", "order", "slot", "active"):
        grp = [t.clone() if isinstance(t, torch.Tensor) else t for t in L.grp]
        slot = L.slot.clone()
        if spoil == "expert":
            grp[2][0] = 8
        elif spoil == "start":
            grp[2][1] = -4
        elif spoil == "count":
            grp[2][2] = 1 << 30
        elif spoil == "order":
            grp[0][0] = 1 << 30
        elif spoil == "slot":
            slot[int(grp[2][0])] = 99
        else:
            grp[1][1] = 1 << 30
        dev = mm16.Moe16Dev(L.dev.gate, L.dev.up, L.dev.down, slot.to(cuda))
        h = marked(cuda, torch.bfloat16, L.P, 32)
        kw = dict(order=grp[0], order_n=grp[1], egrp=grp[2], max_active=grp[3])
        mm16.moe16_gate_up(dev, x, 2, L.P, h, **kw, g=torch.empty_like(h), u=torch.empty_like(h))
        good = marked(cuda, torch.bfloat16, L.P, 32)
        mm16.moe16_gate_up(L.dev, x, 2, L.P, good, **L.kw)
        first = int(L.egrp[2]) if spoil != "order" else 1
        skipped = L.order[:first].long() if spoil != "active" else L.order[:0].long()
        good[skipped] = 77.0
        assert torch.equal(h, good), spoil
        dW = marked(cuda, torch.bfloat16, L.nl, 32, 64)
        mm16.moe16_dw(dev, h, 1, x, 2, L.P, *grp, dW)
        assert not (dW == 77.0).all()
    ids = L.ids_d.clone()
    ids[0], ids[1] = -1, 8
    h = marked(cuda, torch.bfloat16, L.P, 32)
    mm16.moe16_gate_up(L.dev, x, 2, L.P, h, ids=ids)
    assert (h[:2] == 77.0).all() and not (h[2:] == 77.0).all(1).any()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("P,ff", [(1, 8), (3, 33), (7, 768), (130, 1000), (300, 520)])
@pytest.mark.parametrize("clamp", [0.0, 1.5])
def test_swiglu_bwd(cuda, dtype, P, ff, clamp):
    """against the 64-bit formula and, through autograd in 64 bits, its differences' limit; rows that are not listed stay"""
    g = gen(P + ff)
    G, U, D = ((torch.randn(P, ff, generator=g) * 2).to(dtype) for _ in range(3))
    w = torch.rand(P, generator=g)
    gg, uu, ww = G.double().requires_grad_(), U.double().requires_grad_(), w.double().requires_grad_()
    a, b = (gg.clamp_max(clamp), uu.clamp(-clamp, clamp)) if clamp else (gg, uu)
    h = a * torch.sigmoid(a) * b
    (ww[:, None] * h * D.double()).sum().backward()
    on = lambda t: t.to(cuda)  # noqa: E731
    some = torch.randperm(P, generator=g)[:max(1, P - 1)]
    for order in (None, some):
        dg, du, hw = (marked(cuda, dtype, P, ff) for _ in range(3))
        dw = torch.full((P,), 77.0, device=cuda)
        kw = {} if order is None else dict(order=torch.cat([order, order.new_full((P - len(order),), 1 << 30)]).to(torch.int32).to(cuda),
                                           order_n=torch.tensor([len(order), 1], dtype=torch.int32, device=cuda))
        mm16.swiglu_bwd(on(G), on(U), on(D), on(w), dg, du, hw, dw, clamp=clamp, **kw)
        rows = torch.ones(P, dtype=torch.bool) if order is None else torch.zeros(P, dtype=torch.bool).index_fill_(0, order, True)
        r = rows.to(cuda)
        e = 32 * 2.0 ** -24
        within(dg[r], gg.grad[rows], e * (w.double()[:, None] * D.double().abs() * (U.double().abs() + 1))[rows], "dg")
        within(du[r], uu.grad[rows], e * (w.double()[:, None] * D.double().abs() * (G.double().abs() + 1))[rows], "du")
        want = (ww[:, None] * h).detach()
        within(hw[r], want[rows], e * want[rows].abs(), "hw")
        mag = (h.detach().abs() * D.double().abs()).sum(1)
        within(dw[r], ww.grad[rows], ((ff + 32) * 2.0 ** -23 * mag)[rows], "dwts")
        for t in (dg, du, hw, dw):
            assert (t[~r] == 77.0).all()
    dg2, du2 = torch.empty_like(dg), torch.empty_like(du)
    mm16.swiglu_bwd(on(G), on(U), on(D), on(w), dg2, du2, clamp=clamp)
    full = [marked(cuda, dtype, P, ff) for _ in range(2)]
    bufs = [on(G).clone(), on(U).clone(), on(D).clone()]
    mm16.swiglu_bwd(*bufs, on(w), bufs[0], bufs[1], bufs[2], None, clamp=clamp)   # each output over an input
    assert torch.equal(bufs[0], dg2) and torch.equal(bufs[1], du2)


@pytest.mark.parametrize("dtype", TYPES)
def test_rows16(cuda, dtype):
    g = gen(3)
    for m, n, pad in ((1, 1, 0), (5, 64, 0), (7, 37, 3), (130, 1000, 8)):
        x = torch.randn(m, n, generator=g) * 10
        out, ok = empty(m, n, dtype, cuda, pad)
        mm16.rows16(put(x, torch.float32, cuda, pad), out)
        assert torch.equal(out.cpu(), x.to(dtype))
        ok()
    e = torch.tensor([[0.0, -0.0, float("inf"), -float("inf"), NAN, 1e-40, 65519.0, 65520.0, 1 + 2.0 ** -8, 1 + 3 * 2.0 ** -9]])
    out = torch.empty(1, 10, dtype=dtype, device=cuda)
    mm16.rows16(e.to(cuda), out)
    assert torch.equal(out.cpu().view(torch.int16)[~e.isnan()], e.to(dtype).view(torch.int16)[~e.isnan()]) and out[0, 4].isnan()


# ------------------------------------------------------------------ values, places, streams, graphs

@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("m,n,k", [(3, 40, 264), (40, 72, 264), (300, 264, 136)])
def test_infinities_stay_in_their_rows(cuda, dtype, m, n, k):
    g = gen(m)
    W, x = ints(g, n, k, lo=1, hi=3), ints(g, m, k, lo=1, hi=3)
    xi = x.clone()
    xi[0, 5], xi[m - 1, k - 1] = float("inf"), NAN
    out = torch.empty(m, n, dtype=torch.float32, device=cuda)
    mm16.linear(put(W, dtype, cuda, 8), put(xi, dtype, cuda, 8), out)
    same(out, torch.where(torch.tensor([[True]]), xi @ W.t(), xi.new_zeros(1)), "rows with inf and NaN")
    assert (out[0] == float("inf")).all() and out[m - 1].isnan().all() and out[1:m - 1].isfinite().all()
    dW = torch.empty(k, n, dtype=torch.float32, device=cuda)
    dz = ints(g, m, n)
    ws = torch.empty(mm16.linear_dw_ws_bytes(m, k, n), dtype=torch.uint8, device=cuda)
    mm16.linear_dw(put(xi, dtype, cuda, 8), put(dz, dtype, cuda, 8), dW, ws=ws)
    bad = torch.zeros(k, dtype=torch.bool)
    bad[5] = bad[k - 1] = True
    same(dW[(~bad).to(cuda)], (xi[:, ~bad].t() @ dz), "columns without them")


@pytest.mark.parametrize("dtype", [torch.bfloat16])
@pytest.mark.parametrize("m", [3, 20])
def test_rows_beyond_32_bit_offsets(cuda, dtype, m):
    """rows so far apart that byte (and element) offsets pass 2^32"""
    k, n, far = 264, 136, (1 << 33) // m // 8 * 8
    g = gen(m)
    W, x = ints(g, n, k), ints(g, m, k)
    big = torch.empty((m - 1) * far + max(n, k), dtype=dtype, device=cuda)
    xd = big.as_strided((m, k), (far, 1))
    xd.copy_(x.to(dtype))
    out = torch.empty(m, n, dtype=torch.float32, device=cuda)
    mm16.linear(put(W, dtype, cuda), xd, out)
    same(out, x @ W.t(), "far rows of x")
    dW = torch.empty(n, k, dtype=torch.float32, device=cuda)
    dz = ints(g, m, n)
    ws = torch.empty(mm16.linear_dw_ws_bytes(m, n, k), dtype=torch.uint8, device=cuda)
    mm16.linear_dw(put(dz, dtype, cuda), xd, dW, ws=ws)
    same(dW, dz.t() @ x, "far rows in the sum")
    od = big.as_strided((m, n), (far, 1))
    mm16.linear(put(W, dtype, cuda), put(x, dtype, cuda), od)
    same(od, x @ W.t(), "far rows of out")
    w2 = ints(g, m, k)
    xd.copy_(w2.to(dtype))                                     # far rows of W
    x2 = ints(g, 40, k)
    o2 = torch.empty(40, m, dtype=torch.float32, device=cuda)
    mm16.linear(xd, put(x2, dtype, cuda), o2)
    same(o2, x2 @ w2.t(), "far rows of W")
    d2 = ints(g, 40, m)
    o3 = torch.empty(40, k, dtype=torch.float32, device=cuda)
    mm16.linear_dx(xd, put(d2, dtype, cuda), o3)
    same(o3, d2 @ w2, "far rows of W in dx")


def test_broadcast_rows(cuda):
    """one row repeated by a stride of 0"""
    g = gen(8)
    W, x = ints(g, 40, 64), ints(g, 1, 64)
    for m in (3, 50):
        out = torch.empty(m, 40, dtype=torch.float32, device=cuda)
        r = put(ints(g, 1, 40), torch.float32, cuda)
        mm16.linear(put(W, torch.bfloat16, cuda), put(x, torch.bfloat16, cuda).expand(m, 64), out, resid=r.expand(m, 40))
        same(out, (x @ W.t()).expand(m, 40) + r.double().cpu(), "broadcast x")
        dW = torch.empty(40, 64, dtype=torch.float32, device=cuda)
        dz = ints(g, m, 40)
        ws = torch.empty(mm16.linear_dw_ws_bytes(m, 40, 64), dtype=torch.uint8, device=cuda)
        mm16.linear_dw(put(dz, torch.bfloat16, cuda), put(x, torch.bfloat16, cuda).expand(m, 64), dW, ws=ws)
        same(dW, dz.t() @ x.expand(m, 64), "broadcast x in dW")


def _ffn(s):
    """a dense training step and an expert step, as one program makes them"""
    mm16.linear_glu(s["Wg"], s["Wu"], s["x"], s["h"], g=s["g"], u=s["u"])
    mm16.linear(s["Wd"], s["h"], s["y"], resid=s["res"])
    mm16.linear_dx(s["Wd"], s["x"], s["dh"])
    mm16.swiglu_bwd(s["g"], s["u"], s["dh"], s["w"], s["dg"], s["du"], s["hw"], s["dw"])
    mm16.linear_dw(s["dg"], s["x"], s["dWg"], db=s["db"], ws=s["ws"])
    mm16.linear_dx(s["Wg"], s["dg"], s["dx"])
    return s["y"], s["dh"], s["dg"], s["du"], s["hw"], s["dw"], s["dWg"], s["db"], s["dx"]


def _ffn_state(cuda, seed, m=200, d=264, ff=392, dtype=torch.bfloat16):
    g = gen(seed)
    r = lambda *s: (torch.randn(*s, generator=g) * 0.2).to(dtype).to(cuda)  # noqa: E731
    e = lambda *s, dt=dtype: torch.empty(*s, dtype=dt, device=cuda)  # noqa: E731
    return dict(Wg=r(ff, d), Wu=r(ff, d), Wd=r(d, ff), x=r(m, d), res=r(m, d).float(), w=torch.rand(m, generator=g).to(cuda), h=e(m, ff), g=e(m, ff), u=e(m, ff),
                y=e(m, d, dt=torch.float32), dh=e(m, ff), dg=e(m, ff), du=e(m, ff), hw=e(m, ff), dw=e(m, dt=torch.float32),
                dWg=e(ff, d, dt=torch.float32), db=e(ff, dt=torch.float32), dx=e(m, d),
                ws=torch.empty(mm16.linear_dw_ws_bytes(m, ff, d), dtype=torch.uint8, device=cuda))


def test_graphs_and_streams(cuda):
    """the same step eager, on another stream, twice at once on two streams, and replayed from two captured graphs with
    eager work between: the same bits every time"""
    a, b = _ffn_state(cuda, 1), _ffn_state(cuda, 2)
    torch.cuda.synchronize()
    want = [[t.clone() for t in _ffn(s)] for s in (a, b)]
    s1, s2 = torch.cuda.Stream(), torch.cuda.Stream()
    torch.cuda.synchronize()
    for _ in range(3):
        for st, s in ((s1, a), (s2, b)):
            with torch.cuda.stream(st):
                _ffn(s)
        torch.cuda.synchronize()
        for s, w in ((a, want[0]), (b, want[1])):
            out = s["y"], s["dh"], s["dg"], s["du"], s["hw"], s["dw"], s["dWg"], s["db"], s["dx"]
            assert all(torch.equal(p, q) for p, q in zip(out, w))
            for t in out:
                t.zero_()
        torch.cuda.synchronize()
    graphs = []
    for s in (a, b):
        gr = torch.cuda.CUDAGraph()
        with torch.cuda.graph(gr, stream=s1):
            _ffn(s)
        graphs.append(gr)
    for rep in range(4):
        for s, w, gr in zip((a, b), want, graphs):
            x0 = s["x"].clone()
            if rep % 2:
                s["x"].mul_(2)
                again = [t.clone() for t in _ffn(s)]
                gr.replay()
                torch.cuda.synchronize()
                assert all(torch.equal(p, q) for p, q in zip((s["y"], s["dh"], s["dg"], s["du"], s["hw"], s["dw"], s["dWg"], s["db"], s["dx"]), again))
                s["x"].copy_(x0)
            gr.replay()
            torch.cuda.synchronize()
            assert all(torch.equal(p, q) for p, q in zip((s["y"], s["dh"], s["dg"], s["du"], s["hw"], s["dw"], s["dWg"], s["db"], s["dx"]), w)), rep


# ------------------------------------------------------------------ a whole layer

def _layer64(x, W_r, gate, up, down, k, ids, clamp=0.0):
    """the layer in 64 bits for given experts, differentiable: (output, weights)"""
    T = x.shape[0]
    p = torch.softmax(x @ W_r.t(), -1).gather(1, ids)
    w = p / p.sum(1, keepdim=True)
    w = w.detach().requires_grad_()
    out = torch.zeros(T, down.shape[1], dtype=torch.float64)
    for e in range(gate.shape[0]):
        t, j = (ids == e).nonzero(as_tuple=True)
        g, u = x[t] @ gate[e].t(), x[t] @ up[e].t()
        out = out.index_add(0, t, w[t, j][:, None] * ((g * torch.sigmoid(g) * u) @ down[e].t()))
    return out, w


def _rel(a, b):
    return float((a.double().cpu() - b).norm() / b.norm())


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("nt", [1, 2, 5, 40, 300])
@pytest.mark.parametrize("shared", [False, True])
def test_layer_runner(cuda, dtype, nt, shared):
    """router, routing, grouping, experts, combine against 64 bits: inputs and h are rounded to 16 bits (half a step each, so
    at most 4 eps / 2 relative to the sum of magnitudes; the norm of such independent errors stays below 4 eps)"""
    E, d, ff, k = 16, 256, 136, 4
    g = gen(50 + nt)
    r = lambda *s, sc=1.0: torch.randn(*s, generator=g) * sc  # noqa: E731
    gate, up, down = (r(*s, sc=sc).to(dtype) for s, sc in (((E, ff, d), d ** -0.5), ((E, ff, d), d ** -0.5), ((E, d, ff), ff ** -0.5)))
    W_r, x, dy = r(E, d, sc=0.1), r(nt, d), r(nt, d, sc=0.1)
    dev = mm16.Moe16Dev(gate.to(cuda), up.to(cuda), down.to(cuda), torch.arange(E, dtype=torch.int32, device=cuda))
    sh = mm16.Moe16Dev(gate[:1].to(cuda), up[:1].to(cuda), down[:1].to(cuda), torch.zeros(1, dtype=torch.int32, device=cuda)) if shared else None
    run = mm16.Moe16LayerRunner(dev, W_r.to(cuda), k, 300, shared=sh)
    out = run.forward(x.to(cuda)).clone()
    ids = run.ids[:nt * k].view(nt, k).long().cpu()
    leaves = [t.double().requires_grad_() for t in (x.to(dtype), gate, up, down)]
    want, w = _layer64(leaves[0], W_r.double(), *leaves[1:], k, ids)
    S = 0.0
    if shared:
        xs = x.to(dtype).double()
        a = xs @ gate[0].double().t()
        S = (a * torch.sigmoid(a) * (xs @ up[0].double().t())) @ down[0].double().t()
    eps = torch.finfo(dtype).eps
    assert _rel(out, want.detach() + S) < 4 * eps
    kept = run.forward(x.to(cuda), keep=True).clone()
    assert _rel(kept, want.detach() + S) < 4 * eps
    grads = run.backward(dy.to(cuda))
    want.backward(dy.double())
    for name, t in zip(("dx", "gate", "up", "down"), leaves):
        assert _rel(grads[name], t.grad) < 8 * eps, name
    assert _rel(grads["dwts"], w.grad) < 8 * eps
    # a difference of the 64-bit layer along the gradient says the same as its square: the formula that was compared with
    step = 1e-4
    with torch.no_grad():
        moved = [leaves[0]] + [t + step * t.grad for t in leaves[1:]]
        back = [leaves[0]] + [t - step * t.grad for t in leaves[1:]]
        dif = ((_layer64(moved[0], W_r.double(), *moved[1:], k, ids)[0] - _layer64(back[0], W_r.double(), *back[1:], k, ids)[0]) * dy.double()).sum() / (2 * step)
        sq = sum((t.grad ** 2).sum() for t in leaves[1:])
        assert abs(float(dif / sq) - 1) < 1e-3


def test_layer_runner_with_absent_experts_and_captured(cuda):
    E, d, ff, k, nt = 8, 64, 40, 2, 6
    g = gen(9)
    dt = torch.bfloat16
    r = lambda *s: (torch.randn(*s, generator=g) * 0.1).to(dt).to(cuda)  # noqa: E731
    slot = torch.arange(E, dtype=torch.int32)
    slot[3] = -1
    dev = mm16.Moe16Dev(r(E, ff, d), r(E, ff, d), r(E, d, ff), slot.to(cuda))
    run = mm16.Moe16LayerRunner(dev, torch.randn(E, d, generator=g).to(cuda), k, nt)
    run.y.fill_(NAN)
    x = torch.randn(nt, d, generator=g).to(cuda)
    for n in (nt, 1):
        assert run.forward(x[:n]).isfinite().all()
    with pytest.raises(ValueError, match="local"):
        run.forward(x, keep=True)
        run.backward(x)
    with pytest.raises(ValueError):
        run.forward(x.double())
    eager = run.forward(x).clone()
    st = torch.cuda.Stream()
    with torch.cuda.stream(st):
        run.forward(x)
    torch.cuda.synchronize()
    gr = torch.cuda.CUDAGraph()
    with torch.cuda.graph(gr, stream=st):
        out = run.forward(x)
    for _ in range(3):
        run.out.zero_()
        run.y.fill_(NAN)
        gr.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, eager)


@pytest.mark.parametrize("dtype", TYPES)
def test_gguf_experts(cuda, dtype, tmp_path):
    """F16 / BF16 expert tensors of a GGUF file, through the Python reader and through hy_upload_experts: the same rows"""
    import ctypes

    from hyper_amd import check, hy_moe_dev, lib
    from hyper_amd.gguf import GGUF
    from .gguf_writer import STR, U32, write_gguf
    E, d, ff = 3, 72, 40
    g = gen(4)
    gate, up, down = (torch.randn(*s, generator=g).to(dtype) for s in ((E, ff, d), (E, ff, d), (E, d, ff)))
    gt = 1 if dtype == torch.float16 else 30
    raw = lambda t: t.view(torch.int16).numpy().tobytes()  # noqa: E731
    path = str(tmp_path / "m.gguf")
    write_gguf(path, [("general.architecture", STR, "qwen3moe"), ("general.alignment", U32, 32)],
               [("blk.1.ffn_gate_exps.weight", gt, [d, ff, E], raw(gate)), ("blk.1.ffn_up_exps.weight", gt, [d, ff, E], raw(up)),
                ("blk.1.ffn_down_exps.weight", gt, [ff, d, E], raw(down))])
    G = GGUF(path)
    dev = mm16.experts_from_gguf(G, 1, cuda)
    assert torch.equal(dev.gate.cpu(), gate) and torch.equal(dev.up.cpu(), up) and torch.equal(dev.down.cpu(), down)
    t, out = G.expert_tensors(1, E), hy_moe_dev()
    sl = np.array([1, -1, 0], np.int32)
    check(lib().hy_upload_experts(ctypes.byref(t), sl.ctypes.data_as(ctypes.c_void_p), ff, d, 0.0, ctypes.byref(out)))
    x = torch.randn(2, d, generator=g).to(dtype).to(cuda)
    ids = torch.tensor([0, 2, 1, 0], dtype=torch.int32, device=cuda)
    h, h2 = marked(cuda, dtype, 4, ff), marked(cuda, dtype, 4, ff)
    mm16.moe16_gate_up(dev, x, 2, 4, h, ids=ids)
    p = lambda v: ctypes.c_void_p(v.data_ptr())  # noqa: E731
    check(lib().hy_moe16_gate_up(ctypes.byref(out), p(x), d, 2, p(ids), 4, None, None, None, 0, None, None, p(h2),
                                 ctypes.c_void_p(torch.cuda.current_stream().cuda_stream)))
    torch.cuda.synchronize()
    assert torch.equal(h2[[0, 1, 3]], h[[0, 1, 3]]) and (h2[2] == 77.0).all()
    check(lib().hy_free_experts(ctypes.byref(out)))
