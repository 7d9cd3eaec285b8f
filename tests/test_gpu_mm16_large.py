"""16-bit matrix products of the sizes that take the large tiles, against 64-bit products on the device.

All on small integers: every sum is an integer below 2^24 (at most 9 * 4100 here), exact in any order of fp32 sums, so a float32
output equals the formula's bit for bit and a 16-bit output is its nearest value."""
import pytest
import torch

from hyper_amd import mm16
from tests.helpers import gen
from tests.test_gpu_mm16 import TYPES, Layer, empty, glu_err, ints, marked, put, same, within

pytestmark = pytest.mark.gpu


def mul(cuda, a, b):
    """a b^T in 64 bits"""
    return (a.to(cuda) @ b.to(cuda).t().contiguous()).cpu()


# (and few rows: blocks of 16 columns)
# rows and columns that fill many 256 x 256, 128 x 128 and 64 x 128 tiles, none of them whole at the edges; contractions of one
# value, less than a stage of 64, whole stages, and a remainder
DENSE = [(4000, 4000, 520), (4600, 4600, 328), (3900, 4040, 321), (4000, 4104, 520), (4100, 4096, 64), (4090, 3976, 1), (2040, 2056, 264), (1032, 2184, 72), (700, 2056, 136), (257, 8200, 200),
         (64, 8200, 328), (16, 4096, 4096), (3, 4088, 2056), (9, 24, 8200), (40, 8200, 72), (20, 4104, 1032)]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("m,n,k", DENSE)
def test_linear(cuda, dtype, m, n, k):
    g = gen(m + n + k)
    kk = (k + 7) // 8 * 8                                        # whole 16-byte rows, the columns behind k full of NaN
    W, x, b, r = ints(g, n, k), ints(g, m, k), ints(g, 1, n), ints(g, m, n)
    Wd, xd = put(W, dtype, cuda, kk - k), put(x, dtype, cuda, kk - k)
    want = mul(cuda, x, W)
    for out_t in (dtype, torch.float32):
        y, clean = empty(m, n, out_t, cuda, 8)
        z, zclean = empty(m, n, dtype, cuda)
        mm16.linear(Wd, xd, y, bias=b[0].float().to(cuda), act="relu", resid=put(r, out_t, cuda, 16), z=z)
        same(z, want + b, "z")
        same(y, (want + b).clamp_min(0) + r, "y")
        clean(), zclean()
        y, clean = empty(m, n, out_t, cuda)
        mm16.linear(Wd, xd, y)
        same(y, want, "y alone")
        clean()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("m,n,k", [(4000, 2000, 520), (4600, 2304, 328), (4000, 2056, 264), (2040, 1032, 136), (700, 1032, 72), (100, 4104, 264)])
def test_linear_glu(cuda, dtype, m, n, k):
    g = gen(m + n + k)
    Wg, Wu, x = ints(g, n, k, lo=-1, hi=1), ints(g, n, k), ints(g, m, k, lo=-1, hi=1)
    G, U = mul(cuda, x, Wg), mul(cuda, x, Wu)
    outs = [empty(m, n, dtype, cuda) for _ in range(3)]
    mm16.linear_glu(put(Wg, dtype, cuda), put(Wu, dtype, cuda), put(x, dtype, cuda, 8), outs[2][0], g=outs[0][0], u=outs[1][0])
    same(outs[0][0], G, "g")
    same(outs[1][0], U, "u")
    want = G * torch.sigmoid(G) * U
    within(outs[2][0], want, glu_err(want, U), "h")
    for _, clean in outs:
        clean()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("m,n,k", [(520, 4000, 4000), (4000, 520, 3960), (520, 4000, 4104), (64, 4104, 4096), (1, 4096, 3976), (264, 2040, 2056), (4100, 520, 1032), (4000, 1288, 264),
                                   (4104, 264, 4096), (40, 1032, 8200), (1100, 136, 2056),
                                   (8200, 136, 264), (4099, 520, 520), (2048, 1000, 1032), (16400, 8, 8)])
def test_linear_gradients(cuda, dtype, m, n, k):
    """m rows of dz [m, n] and x [m, k]: dx contracts over n, dW and db over m"""
    g = gen(m + n + k)
    W, dz, x = ints(g, n, k), ints(g, m, n), ints(g, m, k)
    Wd, dzd, xd = put(W, dtype, cuda), put(dz, dtype, cuda, 8), put(x, dtype, cuda, 16)
    for out_t in (dtype, torch.float32):
        dx, clean = empty(m, k, out_t, cuda, 8)
        mm16.linear_dx(Wd, dzd, dx)
        same(dx, mul(cuda, dz, W.t()), "dx")
        clean()
        dW, clean = empty(n, k, out_t, cuda)
        db = torch.zeros(n, device=cuda)
        ws = torch.full((mm16.linear_dw_ws_bytes(m, n, k),), 255, dtype=torch.uint8, device=cuda)   # NaN in fp32
        want = mul(cuda, dz.t(), x.t())
        mm16.linear_dw(dzd, xd, dW, db=db, ws=ws)
        same(dW, want, "dW")
        same(db, dz.sum(0), "db")
        dW.fill_(5.0)
        db.fill_(-2.0)
        mm16.linear_dw(dzd, xd, dW, db=db, accumulate=True, ws=ws)
        same(dW, want + 5, "dW accumulated")
        same(db, dz.sum(0) - 2, "db accumulated")
        clean()


class LargeLayer(Layer):
    """the same layer with its formulas evaluated on the device"""

    def __init__(self, cuda, *a, **kw):
        super().__init__(cuda, *a, **kw)
        self.cuda = cuda

    def fwd(self, W, rows):
        out = torch.zeros(self.P, W.shape[1], dtype=torch.float64)
        for e in range(self.nl):
            p = (self.local & (self.le == e)).nonzero().view(-1)
            if len(p):
                out[p] = mul(self.cuda, rows[p], W[e])
        return out

    def dw(self, a, b):
        out = torch.zeros(self.nl, a.shape[1], b.shape[1], dtype=torch.float64)
        for e in range(self.nl):
            p = (self.local & (self.le == e)).nonzero().view(-1)
            if len(p):
                out[e] = mul(self.cuda, a[p].t(), b[p].t())
        return out


# tokens, d, E, k, ff, routing: some 300 rows a group (ends of every length), long and empty groups, about 100, 60 and 20 a group;
# groups that end in whole tiles of 256 rows and in every part of one, about 750 a group;
# one group of more than 1024 pairs among short ones, gradients of six column tiles
GROUPED = [(3000, 2056, 8, 2, 1032, "even"), (2300, 2056, 8, 2, 1032, "skew"), (2400, 520, 16, 2, 2056, "even"), (2300, 264, 8, 2, 1032, "skew"), (1200, 1160, 24, 2, 776, "even"), (500, 1160, 64, 8, 520, "even"),
           (640, 776, 64, 2, 1288, "even"), (1300, 1288, 64, 1, 520, "skew"), (700, 264, 130, 4, 264, "even")]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("T,d,E,k,ff,kind", GROUPED)
@pytest.mark.parametrize("missing", [False, True])
def test_expert_products(cuda, dtype, T, d, E, k, ff, kind, missing):
    L = LargeLayer(cuda, dtype, T, d, E, k, ff, kind, missing)
    loc = L.local
    xp = L.x[L.tok]
    G, U = L.fwd(L.gate, xp), L.fwd(L.up, xp)
    h, g, u = (marked(cuda, dtype, L.P, ff) for _ in range(3))
    mm16.moe16_gate_up(L.dev, put(L.x, dtype, cuda, 8), k, L.P, h, **L.kw, g=g, u=u)
    same(g[loc.to(cuda)], G[loc], "g")
    same(u[loc.to(cuda)], U[loc], "u")
    want = G * torch.sigmoid(G) * U
    within(h[loc.to(cuda)], want[loc], glu_err(want[loc], U[loc]), "h")
    assert (h[~loc.to(cuda)] == 77.0).all()
    hrows = ints(L.g, L.P, ff)
    want = L.fwd(L.down, hrows)
    for out_t, w in ((dtype, L.wts), (torch.float32, None)):
        y = marked(cuda, out_t, L.P, d)
        mm16.moe16_down(L.dev, hrows.to(dtype).to(cuda), L.P, y, wts=None if w is None else w.float().to(cuda), **L.kw)
        same(y[loc.to(cuda)], (want if w is None else want * w[:, None])[loc], f"y {out_t}")
        assert (y[~loc.to(cuda)] == 77.0).all()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("T,d,E,k,ff,kind", GROUPED)
@pytest.mark.parametrize("missing", [False, True])
def test_expert_gradients(cuda, dtype, T, d, E, k, ff, kind, missing):
    L = LargeLayer(cuda, dtype, T, d, E, k, ff, kind, missing, seed=1)
    loc = L.local
    dy, dg, du, hw = ints(L.g, T, d), ints(L.g, L.P, ff), ints(L.g, L.P, ff), ints(L.g, L.P, ff)
    on = lambda t: t.to(dtype).to(cuda)  # noqa: E731
    dyd, dgd, dud, hwd, xd = put(dy, dtype, cuda, 8), on(dg), on(du), on(hw), on(L.x)
    dh = marked(cuda, dtype, L.P, ff)
    mm16.moe16_down_dx(L.dev, dyd, k, L.P, *L.grp, dh)
    same(dh[loc.to(cuda)], L.fwd(L.down.transpose(1, 2), dy[L.tok])[loc], "dh")
    dx = marked(cuda, torch.float32, L.P, d)
    mm16.moe16_gate_up_dx(L.dev, dgd, dud, L.P, *L.grp, dx)
    same(dx[loc.to(cuda)], (L.fwd(L.gate.transpose(1, 2), dg) + L.fwd(L.up.transpose(1, 2), du))[loc], "dx")
    assert (dh[~loc.to(cuda)] == 77.0).all() and (dx[~loc.to(cuda)] == 77.0).all()
    for name, a, ka, A, b, kb, B in (("gate", dgd, 1, dg, xd, k, L.x[L.tok]), ("down", dyd, k, dy[L.tok], hwd, 1, hw)):
        want = L.dw(A, B)
        for out_t in (dtype, torch.float32):
            dW = marked(cuda, out_t, L.nl, *want.shape[1:])
            mm16.moe16_dw(L.dev, a, ka, b, kb, L.P, *L.grp, dW)
            same(dW, want, f"dW {name} {out_t}")
            dW.fill_(3.0)
            mm16.moe16_dw(L.dev, a, ka, b, kb, L.P, *L.grp, dW, accumulate=True)
            same(dW, want + 3, f"dW {name} accumulated {out_t}")


def test_gradients_captured_and_repeated(cuda):
    """experts' gradients and a cut contraction in one captured graph on a stream of its own, replayed on new inputs between eager
    calls: every result is the formula's, the workspace's surroundings stay, and two runs are equal bit for bit"""
    T, d, E, k, ff, m, n = 700, 264, 130, 4, 264, 8200, 136
    L = LargeLayer(cuda, torch.bfloat16, T, d, E, k, ff)
    need = mm16.linear_dw_ws_bytes(m, n, d)
    assert need > 0
    guard = torch.full((need + 64,), 77, dtype=torch.uint8, device=cuda)
    ws = guard[:need]
    dg, x = torch.empty(L.P, ff, dtype=torch.bfloat16, device=cuda), torch.empty(T, d, dtype=torch.bfloat16, device=cuda)
    dz, xs = torch.empty(m, n, dtype=torch.bfloat16, device=cuda), torch.empty(m, d, dtype=torch.bfloat16, device=cuda)
    dW, dE = torch.empty(n, d, device=cuda), torch.empty(L.nl, ff, d, device=cuda)
    db = torch.empty(n, device=cuda)

    def step(stream=None):
        mm16.moe16_dw(L.dev, dg, 1, x, k, L.P, *L.grp, dE, stream=stream)
        mm16.linear_dw(dz, xs, dW, db=db, ws=ws, stream=stream)

    def fill(seed):
        g = gen(seed)
        vals = ints(g, L.P, ff), ints(g, T, d), ints(g, m, n), ints(g, m, d)
        for t, v in zip((dg, x, dz, xs), vals):
            t.copy_(v)
        return L.dw(vals[0], vals[1][L.tok]), mul(cuda, vals[2].t(), vals[3].t()), vals[2].sum(0)

    def check(want):
        for t, w in zip((dE, dW, db), want):
            same(t, w)
            t.fill_(77.0)
        assert (guard[need:] == 77).all()

    want = fill(1)
    step()
    first = dE.clone(), dW.clone()
    check(want)
    step()
    assert torch.equal(first[0], dE) and torch.equal(first[1], dW)
    side = torch.cuda.Stream(cuda)
    side.wait_stream(torch.cuda.current_stream(cuda))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        step(side)
    for seed in (2, 3, 4):
        want = fill(seed)
        torch.cuda.synchronize(cuda)
        graph.replay()
        torch.cuda.synchronize(cuda)
        check(want)
        step()                                                   # eager, on the current stream, between the replays
        torch.cuda.synchronize(cuda)
        check(want)


@pytest.mark.parametrize("out_t", [torch.bfloat16, torch.float32])
def test_gradients_bad_tables(cuda, out_t):
    """pairs that are none and groups outside the pairs add nothing; every gradient is still written"""
    L = LargeLayer(cuda, torch.bfloat16, 700, 264, 130, 4, 264, seed=2)
    a, b = ints(L.g, L.P, L.ff), ints(L.g, L.P, L.d)
    order, egrp = L.order.cpu(), L.egrp.cpu()
    order_bad, egrp_bad = order.clone(), egrp.clone()
    order_bad[0], order_bad[5], order_bad[6] = -1, L.P, 1 << 30
    gone = {int(order[i]) for i in (0, 5, 6)}
    e2, start2, cnt2 = (int(v) for v in egrp[6:9])
    egrp_bad[8] = 1 << 30                                        # the third group: too long
    gone |= {int(p) for p in order[start2:start2 + cnt2]}
    keep = torch.ones(L.P, 1, dtype=torch.float64)
    keep[list(gone)] = 0
    dW = marked(cuda, out_t, L.nl, L.ff, L.d)
    mm16.moe16_dw(L.dev, a.bfloat16().to(cuda), 1, b.bfloat16().to(cuda), 1, L.P, order_bad.to(cuda), L.order_n, egrp_bad.to(cuda), L.ma, dW)
    same(dW, L.dw(a * keep, b))


@pytest.mark.parametrize("pad,offset", [(3, 1), (8, 4), (1, 0)])
def test_outputs_of_any_alignment(cuda, pad, offset):
    """operands on 16 bytes, outputs and what is added to them anywhere: every kernel's last step one element at a time"""
    dtype = torch.bfloat16
    for m, n, k in ((1, 136, 264), (9, 136, 264), (40, 264, 136), (264, 520, 136), (1032, 2184, 72), (4000, 4000, 520), (8200, 136, 264)):
        g = gen(m + n + k + pad)
        W, x, dz, r = ints(g, n, k), ints(g, m, k), ints(g, m, n), ints(g, m, n)
        Wd, xd, dzd = (put(t, dtype, cuda) for t in (W, x, dz))
        b = ints(g, 1, n)[0]
        bd = torch.empty(n + 1, device=cuda)[1:]
        bd.copy_(b)
        want = mul(cuda, x, W) + b
        for out_t in (dtype, torch.float32):
            y, clean = empty(m, n, out_t, cuda, pad, offset)
            z, zclean = empty(m, n, dtype, cuda, pad, offset)
            mm16.linear(Wd, xd, y, bias=bd, act="relu", resid=put(r, out_t, cuda, pad, offset), z=z)
            same(z, want, "z")
            same(y, want.clamp_min(0) + r, "y")
            clean(), zclean()
            dx, clean = empty(m, k, out_t, cuda, pad, offset)
            mm16.linear_dx(Wd, dzd, dx)
            same(dx, mul(cuda, dz, W.t()), "dx")
            clean()
            dW, clean = empty(n, k, out_t, cuda, pad, offset)
            ws = torch.empty(mm16.linear_dw_ws_bytes(m, n, k), dtype=torch.uint8, device=cuda)
            dW.fill_(-4.0)
            mm16.linear_dw(dzd, xd, dW, accumulate=True, ws=ws)
            same(dW, mul(cuda, dz.t(), x.t()) - 4, "dW")
            clean()
        h, clean = empty(m, n, dtype, cuda, pad, offset)
        gk, gclean = empty(m, n, dtype, cuda, pad, offset)
        u, uclean = empty(m, n, dtype, cuda, pad, offset)
        mm16.linear_glu(Wd, Wd, xd, h, g=gk, u=u)
        same(gk, want - b, "g")
        same(u, want - b, "u")
        clean(), gclean(), uclean()


def test_expert_outputs_of_any_alignment(cuda):
    """contiguous outputs that start one element off 16 bytes"""
    dtype = torch.bfloat16
    for T, d, E, k, ff in ((700, 264, 130, 4, 264), (37, 264, 20, 8, 136)):
        L = LargeLayer(cuda, dtype, T, d, E, k, ff, seed=5)
        off = lambda t, *s: torch.full((s[0] * s[1] * (s[2] if len(s) > 2 else 1) + 1,), 77.0, dtype=t, device=cuda)[1:].view(*s)  # noqa: E731
        dy, dg, hw = ints(L.g, T, d), ints(L.g, L.P, ff), ints(L.g, L.P, ff)
        h, g, u = (off(dtype, L.P, ff) for _ in range(3))
        mm16.moe16_gate_up(L.dev, put(L.x, dtype, cuda), k, L.P, h, **L.kw, g=g, u=u)
        same(g, L.fwd(L.gate, L.x[L.tok]), "g")
        same(u, L.fwd(L.up, L.x[L.tok]), "u")
        for out_t in (dtype, torch.float32):
            y, dh, dW = off(out_t, L.P, d), off(out_t, L.P, ff), off(out_t, L.nl, ff, d)
            mm16.moe16_down(L.dev, put(hw, dtype, cuda), L.P, y, **L.kw)
            same(y, L.fwd(L.down, hw), "y")
            mm16.moe16_down_dx(L.dev, put(dy, dtype, cuda), k, L.P, *L.grp, dh)
            same(dh, L.fwd(L.down.transpose(1, 2), dy[L.tok]), "dh")
            mm16.moe16_dw(L.dev, put(dg, dtype, cuda), 1, put(L.x, dtype, cuda), k, L.P, *L.grp, dW)
            same(dW, L.dw(dg, L.x[L.tok]), "dW")
