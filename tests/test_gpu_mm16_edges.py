"""The 16-bit products at the ends of their ranges: many pairs, infinities and NaN, slot tables that change, empty calls.

Products are on small integers, exact in any order of fp32 sums, as in test_gpu_mm16."""
import math

import pytest
import torch

from hyper_amd import mm16, moe
from tests.helpers import gen
from tests.test_gpu_mm16 import TYPES, act64, same

pytestmark = pytest.mark.gpu


def dints(g, dev, *shape, lo=-3, hi=3, dtype=torch.bfloat16):
    return torch.randint(lo, hi + 1, shape, generator=g, device=dev).to(dtype)


@pytest.mark.parametrize("d", [8, 9])   # rows of whole 16-byte pieces, and not
def test_more_than_2_24_tokens(cuda, d):
    """2^24 + 4096 tokens of two pairs: products of a pair's number and a constant pass 64 bits unless they are kept short"""
    T, k, E, ff = 2 ** 24 + 4096, 2, 4, 8
    P = T * k
    g = torch.Generator(device=cuda)
    g.manual_seed(d)
    gate, up, down = dints(g, cuda, E, ff, d), dints(g, cuda, E, ff, d), dints(g, cuda, E, d, ff)
    x, dy = dints(g, cuda, T, d), dints(g, cuda, T, d)
    m = mm16.Moe16Dev(gate, up, down, torch.arange(E, dtype=torch.int32, device=cuda))
    # pair p has expert p % 4
    order = torch.arange(P, dtype=torch.int32, device=cuda).view(-1, E).t().reshape(-1).contiguous()
    egrp = torch.tensor([v for e in range(E) for v in (e, e * (P // E), P // E)], dtype=torch.int32, device=cuda)
    grp = (order, torch.tensor([P, E], dtype=torch.int32, device=cuda), egrp, E)
    tok = [torch.arange(e, P, E, device=cuda) // k for e in range(E)]

    def rows(got, src, W, what):   # got[p] = src[token of p] W_e^T
        for e in range(E):
            want = (src[tok[e]].float() @ W[e].float().t()).to(got.dtype)
            assert torch.equal(got[e::E], want), (what, e)
    h, gg, uu = (torch.empty(P, ff, dtype=torch.bfloat16, device=cuda) for _ in range(3))
    mm16.moe16_gate_up(m, x, k, P, h, order=order, order_n=grp[1], egrp=egrp, max_active=E, g=gg, u=uu)
    rows(gg, x, gate, "g")
    rows(uu, x, up, "u")
    del h, uu
    mm16.moe16_down_dx(m, dy, k, P, *grp, gg)
    rows(gg, dy, down.transpose(1, 2), "dh")
    # the sums over pairs: rows that are not zero at both ends of the range and around token 2^24 (sums up to 9 * 3 * 4096)
    a = torch.zeros(P, ff, dtype=torch.bfloat16, device=cuda)
    for at in (0, 2 ** 25 - 4096, P - 4096):
        a[at:at + 4096] = dints(g, cuda, 4096, ff)
    want = torch.stack([a[e::E].float().t() @ x[tok[e]].float() for e in range(E)])
    dW = torch.empty(E, ff, d, device=cuda)
    mm16.moe16_dw(m, a, 1, x, k, P, *grp, dW)
    assert torch.equal(dW, want), "gate's gradient"
    dW2 = torch.empty(E, d, ff, device=cuda)
    mm16.moe16_dw(m, x, k, a, 1, P, *grp, dW2)
    assert torch.equal(dW2, want.transpose(1, 2)), "rows of tokens on the left"


def ends(dtype):
    """infinities, NaN and both signs of values from nothing to the type's largest"""
    v = [float("inf"), float("nan"), 0.0, 1.0, 5.0, 13.875, 14.5, 30.0, 100.0, 3e4] + ([1e15, 1e20, 1e30, 3e38] if dtype == torch.bfloat16 else [])
    return torch.tensor([s * t for t in v for s in (1.0, -1.0)]).to(dtype)


def agrees(got, want, rel, tiny, what):
    """equal where the formula is infinite or NaN, else within rel of it, or tiny (values whose exponentials leave the normal numbers)"""
    rel, tiny = (torch.as_tensor(v, dtype=torch.float64).expand_as(want) for v in (rel, tiny))
    got = got.double().cpu()
    wild = ~want.isfinite()
    assert torch.equal(got[wild].nan_to_num(nan=7.0), want[wild].nan_to_num(nan=7.0)), (what, got, want)
    off = (got[~wild] - want[~wild]).abs()
    assert (off <= rel[~wild] * want[~wild].abs() + tiny[~wild]).all(), (what, got, want)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("act", list(mm16.ACTS))
@pytest.mark.parametrize("m,k", [(1, 8), (5, 8), (5, 9), (40, 8), (300, 8), (40, 9)])   # each kernel that ends in an activation
def test_activations_of_extreme_values(cuda, dtype, act, m, k):
    """against the formula in 64 bits: it is +inf at +inf, and NaN where it is 0 times an infinity.  Bound: a few 2^-24 of
    evaluation; gelu_tanh's exponent is the result of four roundings, each half a step of an exponent of at most 88, and an
    absolute error of an exponent is a relative one of the value."""
    z = ends(dtype)
    n = z.numel()
    W, x = torch.zeros(n, k, dtype=dtype), torch.zeros(m, k, dtype=dtype)
    W[:, 0], x[:, 0] = z, 1.0
    out = torch.empty(m, n, dtype=torch.float32, device=cuda)
    mm16.linear(W.to(cuda), x.to(cuda), out, act=act)
    rel = 16 * 2.0 ** -24
    if act == "gelu_tanh":
        rel = rel + 4 * 2.0 ** -24 * (1.6 * (z.double() + 0.044715 * z.double() ** 3)).abs().clamp_max(88).nan_to_num()
    agrees(out, act64(act, z.double()).expand(m, n), rel, 1e-36, act)


def act_grad64(name, z):
    if name == "relu":
        return torch.where(z.isnan(), z, (z > 0).double())
    if name == "silu":
        s = torch.sigmoid(z)
        return s + z * s * (1 - s)
    if name == "gelu":
        return 0.5 * torch.erfc(-z / math.sqrt(2)) + z * torch.exp(-z * z / 2) / math.sqrt(2 * math.pi)
    if name == "gelu_tanh":
        c = math.sqrt(2 / math.pi)
        s = torch.sigmoid(2 * c * (z + 0.044715 * z ** 3))
        return s + z * s * (1 - s) * 2 * c * (1 + 0.134145 * z * z)
    return torch.ones_like(z)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("act", list(mm16.ACTS))
@pytest.mark.parametrize("odd", [False, True])
def test_activation_gradients_of_extreme_values(cuda, dtype, act, odd):
    """1 and 0 far from zero, up to the type's largest value, whose square is no float; bounds as for the activations, and the
    sum of two terms that the gradient is"""
    z = ends(dtype)
    z = torch.cat([z, z[:(1 if odd else 8 - z.numel() % 8)]])
    out = torch.empty(1, z.numel(), dtype=dtype, device=cuda)
    mm16.act_bwd(act, z[None].to(cuda), torch.ones_like(z)[None].to(cuda), out)
    want, rel = act_grad64(act, z.double())[None], 32 * 2.0 ** -24 + torch.finfo(dtype).eps / 2
    if act == "gelu_tanh":
        rel = rel + 8 * 2.0 ** -24 * (1.6 * (z.double() + 0.044715 * z.double() ** 3)).abs().clamp_max(88).nan_to_num()[None]
    agrees(out, want, rel, 1e-36 if dtype == torch.bfloat16 else 2.0 ** -25, act)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("m,k", [(1, 8), (5, 8), (40, 8), (300, 8), (40, 9)])   # each kernel that ends in a gated product
@pytest.mark.parametrize("clamp", [0.0, 7.0])
def test_gated_products_of_extreme_values(cuda, dtype, m, k, clamp):
    """every pair of a gate and an up value, against the formula in 64 bits: a limit stops infinities and keeps NaN.  Products
    that 64 bits hold and the type does not are infinite; near its largest value only a rounding decides: those are left out, and
    so is silu(-100), which is 0 in the kernels, times an infinity"""
    z = ends(dtype)
    g, u = z.repeat_interleave(z.numel()), z.repeat(z.numel())
    n = g.numel()
    Wg, Wu, x = torch.zeros(n, k, dtype=dtype), torch.zeros(n, k, dtype=dtype), torch.zeros(m, k, dtype=dtype)
    Wg[:, 0], Wu[:, 0], x[:, 0] = g, u, 1.0
    h, gd, ud = (torch.empty(m, n, dtype=dtype, device=cuda) for _ in range(3))
    mm16.linear_glu(Wg.to(cuda), Wu.to(cuda), x.to(cuda), h, clamp=clamp, g=gd, u=ud)
    same(gd, g.double().expand(m, n), "g")
    same(ud, u.double().expand(m, n), "u")
    a, b = g.double(), u.double()
    if clamp:
        a, b = a.clamp_max(clamp), b.clamp(-clamp, clamp)
    want, top = a * torch.sigmoid(a) * b, torch.finfo(dtype).max
    want = torch.where(want.abs() > 1.01 * top, want.sign() * float("inf"), want)
    keep = ~(want.isfinite() & (want.abs() > 0.99 * top)) & ~((a < -87) & (a > -800) & b.isinf())
    # below g = -87.33 silu is 0, at most 1.04e-36 off, and that times u
    agrees(h[:, keep.to(cuda)], want[keep].expand(m, -1), 32 * 2.0 ** -24 + torch.finfo(dtype).eps / 2,
           (1.04e-36 * b.abs() + (2.0 ** -134 if dtype == torch.bfloat16 else 2.0 ** -25)).nan_to_num(posinf=0)[keep].expand(m, -1), f"clamp {clamp}")


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("ff", [64, 33])
def test_gradients_of_nan_below_a_limit(cuda, dtype, ff):
    """a NaN gate or up value shows in what depends on it and in its row's weight, and nowhere else; u = -2 lies beyond the limit
    1.5, so its gradient is 0 whatever the gate is"""
    P = 4
    g, u, dh = (torch.full((P, ff), v, dtype=dtype, device=cuda) for v in (0.5, -2.0, 1.0))
    w = torch.full((P,), 0.5, device=cuda)

    def call():
        o = [torch.empty(P, ff, dtype=dtype, device=cuda) for _ in range(3)] + [torch.empty(P, device=cuda)]
        mm16.swiglu_bwd(g, u, dh, w, *o, clamp=1.5)
        return o
    u[1, 6] = 1.0
    good = call()
    assert all(t.isfinite().all() for t in good)
    g[1, 5] = g[1, 6] = u[2, 7] = float("nan")
    dg, du, hw, dw = call()
    for t, bad in ((dg, [(1, 5), (1, 6), (2, 7)]), (du, [(1, 6)]), (hw, [(1, 5), (1, 6), (2, 7)])):
        mark = torch.zeros(P, ff, dtype=torch.bool, device=cuda)
        for at in bad:
            mark[at] = True
        assert torch.equal(t.isnan(), mark)
    assert torch.equal(dw.isnan().cpu(), torch.tensor([False, True, True, False]))
    assert torch.equal(dg[0], good[0][0]) and torch.equal(du[0], good[1][0]) and torch.equal(hw[3], good[2][3]) and torch.equal(dw[[0, 3]], good[3][[0, 3]])


# ------------------------------------------------------------------ slot tables

@pytest.mark.parametrize("n", [64, 66, 33])   # rows of 16-byte pieces, and not
@pytest.mark.parametrize("nt,k", [(1, 1), (3, 2), (40, 8), (5, 64)])
@pytest.mark.parametrize("shared", [False, True])
def test_combine_of_local_pairs(cuda, n, nt, k, shared):
    """integers, exact in any order; the rows of absent experts hold NaN"""
    E = 70
    g = gen(n + nt + k)
    y = torch.randint(-9, 10, (nt * k, n), generator=g).float()
    ids = torch.stack([torch.randperm(E, generator=g)[:k] for _ in range(nt)]).reshape(-1).to(torch.int32)
    slot = torch.randint(-1, 9, (E,), generator=g).to(torch.int32)
    slot[slot == 8] = 1 << 20                                   # no matrix of the layer's 8
    ids[::7] = torch.tensor([-1, E, 1 << 30, -(1 << 31)], dtype=torch.int32).repeat(nt * k)[:len(ids[::7])]
    there = (ids >= 0) & (ids < E)
    there &= (slot[ids.long().clamp(0, E - 1)] >= 0) & (slot[ids.long().clamp(0, E - 1)] < 8)
    y[~there] = float("nan")
    want = torch.where(there[:, None], y, torch.zeros(())).view(nt, k, n).sum(1)
    b = torch.zeros(8, 8, n, dtype=torch.bfloat16, device=cuda)
    m = mm16.Moe16Dev(b, b, None, slot.to(cuda))
    sh = torch.randint(-9, 10, (nt, n), generator=g).float() if shared else None
    sg = torch.full((nt,), 0.5) if shared else None
    out = torch.full((nt + 1, n), 77.0, device=cuda)
    mm16.moe16_reduce(m, sh.to(cuda) if shared else None, sg.to(cuda) if shared else None, y.to(cuda), k, out, nt, ids.to(cuda))
    assert torch.equal(out[:nt].cpu(), want + (0.5 * sh if shared else 0)) and (out[nt] == 77.0).all()


class _Runner:
    """a layer whose experts can leave; its buffers are filled with NaN before each call"""

    def __init__(self, cuda, nt, without=()):
        g = gen(11)
        r = lambda *s: (torch.randn(*s, generator=g) * 0.1).to(torch.bfloat16).to(cuda)  # noqa: E731
        E, d, ff, k = 8, 64, 40, 2
        self.gate, self.up, self.down = r(E, ff, d), r(E, ff, d), r(E, d, ff)
        for e in without:
            self.down[e] = 0
        self.slot = torch.arange(E, dtype=torch.int32, device=cuda)
        self.x, self.dy = torch.randn(nt, d, generator=g).to(cuda), torch.randn(nt, d, generator=g).to(cuda)
        W_r = torch.randn(E, d, generator=g).to(cuda)
        self.run = mm16.Moe16LayerRunner(mm16.Moe16Dev(self.gate, self.up, self.down, self.slot), W_r, k, nt)

    def forward(self, **kw):
        for t in (self.run.h, self.run.y, self.run.g, self.run.u):
            if t is not None:
                t.fill_(float("nan"))
        return self.run.forward(self.x, **kw).clone()


@pytest.mark.parametrize("nt", [1, 2, 20, 300])
def test_runner_reads_the_slot_table_each_time(cuda, nt):
    """an expert that leaves after the runner was made adds nothing: as one whose down matrix is zeros; the next call has it
    again.  Eager and replayed."""
    full, R = _Runner(cuda, nt), _Runner(cuda, nt)
    want = full.forward()
    gone = _Runner(cuda, nt, without=(2, 3, 5)).forward()
    assert not torch.equal(want, gone) or nt < 20
    assert torch.equal(R.forward(), want)
    out_of = torch.tensor([0, 1, -1, 8, 4, 1 << 30, 6, 7], dtype=torch.int32, device=cuda)
    back = torch.arange(8, dtype=torch.int32, device=cuda)
    R.slot.copy_(out_of)
    assert torch.equal(R.forward(), gone)
    st = torch.cuda.Stream()
    torch.cuda.synchronize()
    gr = torch.cuda.CUDAGraph()
    with torch.cuda.graph(gr, stream=st):
        out = R.run.forward(R.x)
    for table, w in ((back, want), (out_of, gone), (back, want)):
        R.slot.copy_(table)
        R.run.y.fill_(float("nan"))
        R.run.h.fill_(float("nan"))
        torch.cuda.synchronize()
        gr.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, w)
        assert torch.equal(R.forward(), w)


@pytest.mark.parametrize("nt", [1, 20, 300])
def test_runner_backward_with_the_slot_table_of_its_forward(cuda, nt):
    """experts that are away in forward have no part in the gradients and get zeros; tables that change between the two passes
    change nothing.  Against experts whose down matrix is zeros, which only differ in that matrix's own gradient."""
    R, Z = _Runner(cuda, nt), _Runner(cuda, nt, without=(2, 5))
    Z.forward(keep=True)
    want = Z.run.backward(Z.dy)
    for e in (2, 5):
        want["down"][e] = 0
    R.forward(keep=True)
    R.slot[2] = -1
    R.slot[5] = 8
    R.forward(keep=True)
    for change in (None, (2, 2), (0, -1), (slice(None), -1)):
        if change:
            R.slot[change[0]] = change[1]
        got = R.run.backward(R.dy)
        for name, w in want.items():
            assert torch.equal(got[name], w), (name, change)


# T, d, E, experts that share a matrix, k, ff: the element-wise kernel, tiles by pairs, blocks that go through a group's tiles, long groups
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("T,d,E,same_as,k,ff", [(9, 33, 6, {4: 1}, 2, 17), (40, 72, 8, {5: 0, 6: 0, 7: 2}, 3, 40), (700, 136, 5, {3: 2}, 2, 264), (700, 264, 130, {7: 3, 129: 3, 64: 65}, 4, 264),
                                                (2000, 264, 130, {e: 1 for e in range(2, 60)}, 4, 264), (3000, 72, 3, {1: 0, 2: 0}, 2, 40)])
def test_weight_gradients_of_shared_matrices(cuda, dtype, T, d, E, same_as, k, ff):
    """experts that share a local matrix: its gradient is the sum over the pairs of them all, the same every time"""
    g = gen(T + E)
    slot = torch.full((E,), -1, dtype=torch.int32)
    nl = 0
    for e in range(E):
        if e not in same_as:
            slot[e], nl = nl, nl + 1
    for e, o in same_as.items():
        slot[e] = slot[o]
    P = T * k
    ids = torch.stack([torch.randperm(E, generator=g)[:k] for _ in range(T)]).reshape(-1).to(torch.int32)
    r = lambda *s: torch.randint(-3, 4, s, generator=g).to(dtype)  # noqa: E731
    a, b, w = r(P, ff), r(T, d), torch.zeros(nl, ff, d, dtype=dtype, device=cuda)
    m = mm16.Moe16Dev(w, w, None, slot.to(cuda))
    i32 = dict(dtype=torch.int32, device=cuda)
    order, order_n, egrp = torch.zeros(P, **i32), torch.zeros(2, **i32), torch.zeros(3 * E, **i32)
    moe.moe_order(m, ids.to(cuda), P, E, order, order_n, None, egrp)
    le, tok = slot[ids.long()].long(), torch.arange(P) // k
    want = torch.zeros(nl, ff, d, dtype=torch.float64)
    for e in range(nl):
        p = (le == e).nonzero().view(-1)
        want[e] = a[p].double().t() @ b[tok[p]].double()
    for out_t in (torch.float32, dtype):
        dW = torch.full((nl, ff, d), 77.0, dtype=out_t, device=cuda)
        mm16.moe16_dw(m, a.to(cuda), 1, b.to(cuda), k, P, order, order_n, egrp, min(E, P), dW)
        same(dW, want, f"{out_t}")
        again = torch.empty_like(dW)
        mm16.moe16_dw(m, a.to(cuda), 1, b.to(cuda), k, P, order, order_n, egrp, min(E, P), again)
        assert torch.equal(again, dW)


# ------------------------------------------------------------------ empty calls

@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("E,d,ff", [(3, 33, 17), (3, 64, 40), (130, 264, 264), (5, 520, 520)])
def test_no_pairs(cuda, dtype, E, d, ff):
    """empty tensors, a grouping of no entries: outputs of no rows, and gradients of zeros for every expert"""
    e = lambda *s, dt=dtype: torch.empty(*s, dtype=dt, device=cuda)  # noqa: E731
    w = torch.zeros(E, ff, d, dtype=dtype, device=cuda)
    m = mm16.Moe16Dev(w, w, w.view(E, d, ff), torch.arange(E, dtype=torch.int32, device=cuda))
    none = e(0, dt=torch.int32)
    for grp in ((none, none, none, 0), (none, torch.zeros(2, dtype=torch.int32, device=cuda), torch.zeros(3 * E, dtype=torch.int32, device=cuda), E)):
        kw = dict(order=grp[0], order_n=grp[1], egrp=grp[2], max_active=grp[3])
        mm16.moe16_gate_up(m, e(0, d), 2, 0, e(0, ff), **kw)
        mm16.moe16_gate_up(m, e(0, d), 2, 0, e(0, ff), ids=none)
        mm16.moe16_down(m, e(0, ff), 0, e(0, d), **kw)
        mm16.moe16_down(m, e(0, ff), 0, e(0, d), ids=none)
        mm16.moe16_down_dx(m, e(0, d), 2, 0, *grp, e(0, ff))
        mm16.moe16_gate_up_dx(m, e(0, ff), e(0, ff), 0, *grp, e(0, d))
        mm16.swiglu_bwd(e(0, ff), e(0, ff), e(0, ff), None, e(0, ff), e(0, ff), e(0, ff), e(0, dt=torch.float32))
        mm16.moe16_reduce(m, None, None, e(0, d, dt=torch.float32), 2, e(0, d, dt=torch.float32), 0, none)
        for out_t in (dtype, torch.float32):
            buf = torch.full((E * ff * d + 8,), 5.0, dtype=out_t, device=cuda)
            dW = buf[:E * ff * d].view(E, ff, d)
            mm16.moe16_dw(m, e(0, ff), 1, e(0, d), 2, 0, *grp, dW, accumulate=True)
            assert (buf == 5.0).all()
            mm16.moe16_dw(m, e(0, ff), 1, e(0, d), 2, 0, *grp, dW)
            assert (dW == 0).all() and (buf[E * ff * d:] == 5.0).all()


def test_runner_without_rows(cuda):
    """a step of no rows has gradients: zeros.  They belong to the last forward, which kept something or not"""
    R = _Runner(cuda, 20)
    with pytest.raises(ValueError, match="follows"):
        R.run.backward(R.dy[:0])
    for before in (False, True):
        if before:
            R.forward(keep=True)
        assert R.run.forward(R.x[:0], keep=True).shape == (0, 64)
        got = R.run.backward(R.dy[:0])
        assert got["dx"].shape == (0, 64) and got["dwts"].shape == (0, 2)
        for name, t in (("gate", R.gate), ("up", R.up), ("down", R.down)):
            assert got[name].shape == t.shape and (got[name] == 0).all()
        with pytest.raises(ValueError, match="follows"):
            R.run.backward(R.dy)
        R.run.forward(R.x[:0])
        with pytest.raises(ValueError, match="follows"):
            R.run.backward(R.dy[:0])
    R.forward(keep=True)
    first = R.run.backward(R.dy)
    R.forward(keep=True)
    again = R.run.backward(R.dy)
    assert all(torch.equal(first[n], again[n]) for n in first)


def test_overlapping_groups(cuda):
    """1024 groups that each claim all of 2^22 pairs, as no grouping makes them: more tiles than the scan over the groups counts.
    Every block still takes a tile of one of them: with the same weights for all experts, the formula or what was there."""
    T, k, E, d, ff = 1 << 16, 64, 1024, 7, 544
    P = T * k
    g = torch.Generator(device=cuda)
    g.manual_seed(5)
    W = [dints(g, cuda, 1, ff, d).repeat(E, 1, 1) for _ in range(2)]
    x = dints(g, cuda, T, d)
    m = mm16.Moe16Dev(W[0], W[1], None, torch.arange(E, dtype=torch.int32, device=cuda))
    order = torch.arange(P, dtype=torch.int32, device=cuda)
    egrp = torch.stack([torch.arange(E), torch.zeros(E, dtype=torch.long), torch.full((E,), P)], 1).reshape(-1).to(torch.int32).to(cuda)
    buf = torch.full(((P + 2) * ff,), 77.0, dtype=torch.bfloat16, device=cuda)
    h = buf[ff:-ff].view(P, ff)
    mm16.moe16_gate_up(m, x, k, P, h, order=order, order_n=torch.tensor([P, E], dtype=torch.int32, device=cuda), egrp=egrp, max_active=E)
    want = torch.empty(T, ff, dtype=torch.bfloat16, device=cuda)
    mm16.linear_glu(W[0][0], W[1][0], x, want)
    wrong = int(((h.view(T, k, ff) != want[:, None]) & (h.view(T, k, ff) != 77.0)).sum())
    around = int((buf[:ff] != 77.0).sum()) + int((buf[-ff:] != 77.0).sum())
    assert wrong == 0 and around == 0 and bool((h[0] != 77.0).any())
