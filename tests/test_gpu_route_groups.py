"""Routing with groups of experts and its gradient against the formula in 64 bits: the same experts in the same order, the weights
its nearest float32 values (64-bit scores are good to 1e-14, and their order is the formula's unless two lie closer than that).

Two groups whose worths are the same number in exact arithmetic, though not of the same scores and biases (a + (b + t) beside
(a + t) + b), have no order in 64 bits either: a score is off by up to 4 2^-53 of itself (exp, its sum, the quotient), bias and
group sum round by 2^-53 of theirs, on both sides of the comparison.  Such groups, nearer than 16 2^-53 of the terms' sizes, may
come either way; the experts are then those of one of the orders."""
import itertools

import pytest
import torch

from hyper_amd import mm16
from tests.helpers import gen
from tests.test_gpu_mm16 import empty, within

pytestmark = pytest.mark.gpu
INF = float("inf")


def scores64(l, score):
    l = l.double()
    if score == "sigmoid":
        return torch.sigmoid(l)
    return torch.softmax(l, 1)


def best64(v, k):
    """stable: the lower index first among equals"""
    return torch.sort(v, dim=1, descending=True, stable=True).indices[:, :k]


def route64(l, k, score, bias=None, n_group=1, top_group=1, group_best=1, renorm=True, scale=1.0, keep=None):
    """keep: groups given [nt, n_group] instead of the best ones"""
    nt, E = l.shape
    s = scores64(l, score)
    c = s if bias is None else s + bias.double()
    c = torch.where((l.double() > -INF) & (c > -INF), c, torch.full_like(c, -INF))   # (NaN fails too)
    if top_group < n_group:
        by = c.view(nt, n_group, -1)
        top = torch.sort(by, dim=2, descending=True).values[:, :, :group_best]
        worth = torch.where((top > -INF).all(2), top.sum(2), torch.full_like(top[:, :, 0], -INF))
        if keep is None:
            keep = torch.zeros(nt, n_group, dtype=torch.bool).scatter_(1, best64(worth, top_group), True) & (worth > -INF)
        c = torch.where(keep.repeat_interleave(E // n_group, 1), c, torch.full_like(c, -INF))
    ids = best64(c, k)
    on = c.gather(1, ids) > -INF
    z = torch.where(on, s.gather(1, ids), torch.zeros((), dtype=torch.float64))
    if renorm:
        if score == "softmax":
            z = torch.where(on, torch.softmax(torch.where(on, l.double().gather(1, ids), torch.full_like(z, -INF)), 1), torch.zeros_like(z))
        else:
            S = z.sum(1, keepdim=True)
            z = torch.where(S > 0, z / S, torch.zeros_like(z))
    return torch.where(on, ids, torch.full_like(ids, -1)).to(torch.int32), z * scale


def other_orders(l, score, bias, n_group, top_group, group_best):
    """of one token [1, E]: the sets of groups that the orders of equal worths allow"""
    s = scores64(l, score)
    by = (s if bias is None else s + bias.double()).view(n_group, -1)
    top = torch.sort(by, dim=1, descending=True).values[:, :group_best]
    worth, size = top.sum(1), top.abs().sum(1) + 1
    edge = torch.sort(worth, descending=True).values[top_group - 1]
    near = (worth - edge).abs() <= 16 * 2.0 ** -53 * size
    sure = [g for g in range(n_group) if worth[g] > edge and not near[g]]
    for some in itertools.combinations([g for g in range(n_group) if near[g]], top_group - len(sure)):
        keep = torch.zeros(1, n_group, dtype=torch.bool)
        keep[0, sure + list(some)] = True
        yield keep


def check(l, k, dev, ls=0, **how):
    nt, E = l.shape
    if ls:
        wide = torch.full((nt, ls), float("nan"))
        wide[:, :E] = l
        on = wide.to(dev)[:, :E]
    else:
        on = l.to(dev)
    bias = how.get("bias")
    ids, wts = torch.full((nt + 1, k), 77, dtype=torch.int32, device=dev), torch.full((nt + 1, k), 77.0, device=dev)
    mm16.route_groups(on, ids[:nt], wts[:nt], **{**how, "bias": None if bias is None else bias.to(dev)})
    want, w = route64(l, k, **{"score": "softmax", **how})
    got = ids[:nt].cpu()
    full = {"score": "softmax", "bias": None, "n_group": 1, "top_group": 1, "group_best": 1, **how}
    if full["bias"] is not None and full["group_best"] == 2 and full["top_group"] < full["n_group"]:
        for i in (got != want).any(1).nonzero()[:, 0].tolist():
            for keep in other_orders(l[i:i + 1], *(full[n] for n in ("score", "bias", "n_group", "top_group", "group_best"))):
                other, ow = route64(l[i:i + 1], k, **{**full, "keep": keep})
                if torch.equal(other[0], got[i]):
                    want[i], w[i] = other[0], ow[0]
    assert torch.equal(got, want), (how, (got != want).nonzero()[:3].tolist(), got[(got != want).any(1)][:1], want[(got != want).any(1)][:1])
    within(wts[:nt], w, 1e-12 * w.abs() + 1e-30, str(how))
    assert (ids[nt] == 77).all() and (wts[nt] == 77).all()
    return got


def logits(g, nt, E, coarse=False):
    l = 1.5 * torch.randn(nt, E, generator=g)
    return l.to(torch.bfloat16).float() if coarse else l


@pytest.mark.parametrize("E,G", [(1, 1), (2, 1), (2, 2), (16, 4), (60, 6), (63, 1), (64, 8), (65, 5), (96, 48), (128, 8), (160, 8), (256, 8), (256, 64),
                                 (288, 9), (384, 8), (512, 16), (1000, 8), (1024, 64), (1024, 2)])
@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
def test_route_groups_shapes(E, G, score):
    dev = torch.device("cuda:0")
    g = gen(E * 131 + G)
    gs = E // G
    for i, nt in enumerate((1, 5, 130)):
        for T in {1, (G + 1) // 2, G}:
            for best in ((1, 2) if gs > 1 else (1,)):
                k = min(8 if i else 3, gs * T)
                check(logits(g, nt, E, coarse=i == 1), k, dev, score=score, bias=0.05 * torch.randn(E, generator=g) if (i + T) % 2 else None, n_group=G,
                      top_group=T, group_best=best, renorm=(i + best) % 2 == 0, scale=(1.0, 2.5)[best - 1], ls=E + 3 if i == 2 else 0)


@pytest.mark.parametrize("k", [1, 2, 13, 63, 64])
def test_route_groups_of_many(k):
    dev = torch.device("cuda:0")
    for E, G, T in ((64, 1, 1), (128, 2, 1), (1024, 8, 3)):
        check(logits(gen(k + E), 40, E), k, dev, score="sigmoid", n_group=G, top_group=T, renorm=False)


def test_route_groups_ties():
    """equal scores, near and at every border: more of them than a wave has lanes, whole equal groups, few distinct values"""
    dev = torch.device("cuda:0")
    g = gen(3)
    for E, G, T, best in ((1024, 8, 4, 2), (256, 8, 3, 1), (128, 1, 1, 1), (512, 64, 20, 2)):
        for k in (1, 8, 50):
            equal = torch.zeros(3, E)
            equal[1] = -2.5
            equal[2, ::2] = 1.0
            few = torch.randint(0, 3, (64, E), generator=g).float()
            for score in ("softmax", "sigmoid"):
                check(torch.cat([equal, few]), k, dev, score=score, n_group=G, top_group=T, group_best=best)
                check(torch.cat([equal, few]), k, dev, score=score, n_group=G, top_group=T, group_best=best, bias=torch.randint(0, 2, (E,), generator=g).float())


def test_route_groups_near_ties():
    """scores that differ in bits a float32 does not hold: neighbouring logits, a bias that leads and trails the score's difference"""
    dev = torch.device("cuda:0")
    base = torch.full((200, 128), 0.7) + torch.randn(200, 1, generator=gen(8))
    step = torch.randint(-4, 5, (200, 128), generator=gen(9)).float() * 2.0 ** -23
    l = base * (1 + step)
    for score in ("softmax", "sigmoid"):
        check(l, 8, dev, score=score)
        check(l, 8, dev, score=score, n_group=8, top_group=2, group_best=2, bias=torch.randint(-2, 3, (128,), generator=gen(10)).float() * 2.0 ** -26)


def test_route_groups_masks():
    """logits of -inf: experts that may not be chosen, down to rows without any; NaN and +inf"""
    dev = torch.device("cuda:0")
    for score in ("softmax", "sigmoid"):
        l = logits(gen(4), 40, 64)
        for t in range(20):
            l[t, torch.randperm(64, generator=gen(t))[:min(64, 44 + t)]] = -INF
        l[20], l[21, 5:] = -INF, -INF
        l[22, 3] = float("nan")
        l[23], l[24, 9] = float("nan"), INF
        for G, T, best in ((1, 1, 1), (8, 4, 1), (8, 4, 2)):
            for renorm in (True, False):
                ids = check(l, 8, dev, score=score, n_group=G, top_group=T, group_best=best, renorm=renorm)
                assert (ids[20] == -1).all()
        bias = torch.zeros(64)
        bias[::3], bias[1] = -INF, float("nan")
        ids = check(logits(gen(6), 40, 64), 8, dev, score=score, bias=bias)
        assert not ((ids % 3 == 0) | (ids == 1)).any()


def test_route_groups_extreme_logits():
    dev = torch.device("cuda:0")
    l = logits(gen(7), 8, 96)
    l[0] *= 3e4   # one probability is 1, the others underflow in 64 bits too
    l[1] = -800.0 - torch.arange(96)   # sigmoids of 0: no sum to renormalise by
    l[2] = 30 + 0.1 * torch.arange(96)
    l[3] = -3e38
    check(l, 6, dev, score="sigmoid")
    check(l[1:], 6, dev, score="softmax")
    check(l[1:], 6, dev, score="softmax", renorm=False)


# ------------------------------------------------------------------ gradient

def weights64(l, ids, score, renorm, scale):
    """the weights of given experts as a differentiable 64-bit function (ids of -1: weight 0)"""
    on = ids >= 0
    at = ids.long().clamp_min(0)
    if score == "softmax" and renorm:
        z = torch.where(on, l.gather(1, at), torch.full_like(l.gather(1, at), -1e300))
        return torch.where(on, torch.softmax(z, 1), torch.zeros_like(z)) * scale
    s = torch.softmax(l, 1) if score == "softmax" else torch.sigmoid(l)
    z = torch.where(on, s.gather(1, at), torch.zeros_like(s.gather(1, at)))
    if renorm:
        z = z / z.sum(1, keepdim=True).clamp_min(1e-300)
    return z * scale


@pytest.mark.parametrize("dt", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("score,renorm", [("softmax", True), ("softmax", False), ("sigmoid", True), ("sigmoid", False)])
def test_route_groups_bwd(score, renorm, dt):
    dev = torch.device("cuda:0")
    for E, k, nt in ((1, 1, 3), (16, 2, 1), (63, 5, 7), (128, 8, 130), (256, 8, 33), (384, 6, 9), (512, 10, 40), (1000, 64, 5), (1024, 3, 6)):
        g = gen(E + k)
        l = logits(g, nt, E)
        ids = torch.stack([torch.randperm(E, generator=g)[:k] for _ in range(nt)]).to(torch.int32)
        if nt > 4:
            ids[1, 0], ids[2] = -1, -1
            ids[3, k - 1] = E   # outside: takes no part
        dw = torch.randn(nt, k, generator=g)
        x = l.double().requires_grad_()
        known = torch.where(ids < E, ids, torch.full_like(ids, -1))
        weights64(x, known, score, renorm, 2.5).backward(dw.double())
        out, around = empty(nt, E, dt, dev, pad=3)
        wide = torch.full((nt, E + 2), float("nan"))
        wide[:, :E] = l
        mm16.route_groups_bwd(wide.to(dev)[:, :E], ids.to(dev), dw.to(dev), out, score=score, renorm=renorm, scale=2.5)
        # 64-bit arithmetic rounded once to 32 bits (and once more to dt); where terms cancel, 1e-13 of their sizes is left
        size = x.grad.abs()
        within(out, x.grad, 2.0 ** -24 * size + 1e-12, f"{E} {k} {nt}")
        around()
        assert (out.cpu()[2] == 0).all() if nt > 4 else True


def test_route_groups_bwd_of_masked_and_repeated_experts():
    """-inf logits have no gradient; an expert that ids names twice gets both places' gradients"""
    dev = torch.device("cuda:0")
    for score in ("softmax", "sigmoid"):
        for renorm in (True, False):
            l = logits(gen(2), 4, 70)
            l[0, 10:] = -INF
            l[1] = -INF
            ids = torch.tensor([[3, 4, -1], [-1, -1, -1], [5, 5, 9], [0, 69, 1]], dtype=torch.int32)
            dw = torch.randn(4, 3, generator=gen(1))
            rows = [0, 2, 3]
            x = l[rows].double().clamp_min(-1e300).requires_grad_()
            weights64(x, ids[rows], score, renorm, 1.0).backward(dw[rows].double())
            out = torch.empty(4, 70, device=dev)
            mm16.route_groups_bwd(l.to(dev), ids.to(dev), dw.to(dev), out, score=score, renorm=renorm)
            within(out[rows], x.grad, 2.0 ** -23 * x.grad.abs() + 1e-12, score)
            assert (out[1] == 0).all() and (out[0, 10:] == 0).all()


@pytest.mark.parametrize("score,renorm", [("softmax", True), ("softmax", False), ("sigmoid", True), ("sigmoid", False)])
def test_route_groups_gradient_is_the_forward_passs(score, renorm):
    """against central differences of the 64-bit forward pass with its own choice: step 1e-4, error 1e-8 times third derivatives of
    at most 1 a weight, and the gradients' rounding"""
    dev = torch.device("cuda:0")
    g = gen(12)
    l, bias, k = logits(g, 10, 64), 0.05 * torch.randn(64, generator=g), 6
    how = dict(score=score, bias=bias, n_group=8, top_group=4, group_best=2, renorm=renorm, scale=2.0)
    ids, wts = torch.empty(10, k, dtype=torch.int32, device=dev), torch.empty(10, k, device=dev)
    mm16.route_groups(l.to(dev), ids, wts, **{**how, "bias": bias.to(dev)})
    dw, dl = torch.randn(10, k, generator=g), torch.empty(10, 64, device=dev)
    mm16.route_groups_bwd(l.to(dev), ids, dw.to(dev), dl, score=score, renorm=renorm, scale=2.0)
    for i in range(6):
        v = torch.randn(10, 64, generator=g).double()
        hi, lo = (weights64(l.double() + h * v, ids.cpu(), score, renorm, 2.0) for h in (1e-4, -1e-4))
        diff = ((hi - lo) * dw.double()).sum(1) / 2e-4
        got = (dl.double().cpu() * v).sum(1)
        assert ((got - diff).abs() <= 1e-6 + 2.0 ** -22 * (dl.double().cpu() * v).abs().sum(1)).all(), (i, got - diff)


def test_route_groups_captured_replayed_and_on_another_stream():
    dev = torch.device("cuda:0")
    nt, E, k = 200, 256, 8
    how = dict(score="sigmoid", n_group=8, top_group=4, group_best=2, scale=2.5)
    l, bias, dw = torch.empty(nt, E, device=dev), 0.05 * torch.randn(E, generator=gen(1)).to(dev), torch.randn(nt, k, generator=gen(2)).to(dev)

    def buffers():
        return torch.empty(nt, k, dtype=torch.int32, device=dev), torch.empty(nt, k, device=dev), torch.empty(nt, E, dtype=torch.bfloat16, device=dev)

    def step(o, stream=None):
        mm16.route_groups(l, o[0], o[1], bias=bias, stream=stream, **how)
        mm16.route_groups_bwd(l, o[0], dw, o[2], score="sigmoid", scale=2.5, stream=stream)
    a, b, c = buffers(), buffers(), buffers()
    l.copy_(logits(gen(20), nt, E))
    step(b)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step(b)
    for seed in range(4):
        l.copy_(logits(gen(30 + seed), nt, E))
        step(a)
        torch.cuda.synchronize()
        graph.replay()
        s = torch.cuda.Stream()
        torch.cuda.synchronize()
        step(c, s)
        s.synchronize()
        for p, q, r in zip(a, b, c):
            assert torch.equal(p, q) and torch.equal(p, r)


def test_route_groups_without_groups_agrees_with_the_plain_router():
    """one group, softmax, renormalised: what moe_route computes in 32 bits -- the same experts where their probabilities lie apart"""
    from hyper_amd import moe
    dev = torch.device("cuda:0")
    nt, E, k = 64, 128, 8
    l = torch.stack([torch.randperm(E, generator=gen(i)) for i in range(nt)]).float() * 0.05
    ids, wts, i2, w2 = (torch.empty(nt, k, dtype=d, device=dev) for d in (torch.int32, torch.float32, torch.int32, torch.float32))
    mm16.route_groups(l.to(dev), ids, wts)
    moe.moe_route(l.to(dev), E, E, k, i2, w2, None, nt)
    assert torch.equal(ids, i2) and (wts - w2).abs().max() < 1e-6
