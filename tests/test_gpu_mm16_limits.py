"""The SwiGLU limit through the experts' calls and the layer runner, and the activation's gradient written over its inputs."""
import itertools
import math

import pytest
import torch

from hyper_amd import mm16
from tests.helpers import gen
from tests.test_gpu_mm16 import TYPES, Layer, _rel, glu_err, marked, put, same_rows, within

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("P,ff", [(3, 33), (130, 264)])
@pytest.mark.parametrize("clamp", [0.0, 1.5])
def test_swiglu_bwd_over_its_inputs(cuda, dtype, P, ff, clamp):
    """dg, du and hw over g, u and dh in every order, and two of them beside: the bits of separate outputs"""
    g = gen(P)
    src = [(torch.randn(P, ff, generator=g) * 2).to(dtype).to(cuda) for _ in range(3)]
    w = torch.rand(P, generator=g).to(cuda)
    want, wdw = [torch.empty_like(t) for t in src], torch.empty(P, device=cuda)
    mm16.swiglu_bwd(*src, w, *want, wdw, clamp=clamp)
    assert all(t.isfinite().all() for t in want) and (want[2] != 0).any()
    for perm in itertools.permutations(range(3)):
        for inside in ((0, 1, 2), (0,), (1,), (2,), (0, 2)):   # which outputs lie over an input
            bufs, dw = [t.clone() for t in src], torch.empty(P, device=cuda)
            out = [bufs[perm[i]] if i in inside else torch.empty_like(want[i]) for i in range(3)]
            mm16.swiglu_bwd(*bufs, w, *out, dw, clamp=clamp)
            assert all(torch.equal(a, b) for a, b in zip(out, want)) and torch.equal(dw, wdw), (perm, inside)


# by ids and grouped: single rows, small tiles, element-wise, large tiles
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("T,d,E,k,ff", [(1, 64, 8, 2, 32), (3, 33, 4, 1, 17), (37, 264, 20, 8, 136), (700, 136, 3, 2, 520)])
@pytest.mark.parametrize("missing", [False, True])
def test_expert_products_with_a_limit(cuda, dtype, T, d, E, k, ff, missing):
    clamp = 5.0
    L = Layer(cuda, dtype, T, d, E, k, ff, "even", missing, clamp=clamp)
    xp, xd = L.x[L.tok], put(L.x, dtype, cuda)
    G, U = L.fwd(L.gate, xp), L.fwd(L.up, xp)
    assert (G > clamp).any() and (U > clamp).any() and (U < -clamp).any() or T == 1
    a, b = G.clamp_max(clamp), U.clamp(-clamp, clamp)
    want, loc = a * torch.sigmoid(a) * b, L.local
    for how in ((L.kw, dict(ids=L.ids_d)) if T <= 9 else (L.kw,)):
        h, g, u = (marked(cuda, dtype, L.P, ff) for _ in range(3))
        mm16.moe16_gate_up(L.dev, xd, k, L.P, h, **how, g=g, u=u)
        same_rows(g, G, loc, "g, not limited")
        same_rows(u, U, loc, "u, not limited")
        within(h[loc.to(cuda)], want[loc], glu_err(want[loc], b[loc]), "h")
        assert (h[~loc.to(cuda)] == 77.0).all()


def _layer(x, W_r, gate, up, down, k, ids, clamp):
    """the layer in 64 bits with its limit, differentiable: (output, routing weights, how many gates and ups lie beyond)"""
    p = torch.softmax(x @ W_r.t(), -1).gather(1, ids)
    w = (p / p.sum(1, keepdim=True)).detach().requires_grad_()
    out, beyond = torch.zeros(x.shape[0], down.shape[1], dtype=torch.float64), 0
    for e in range(gate.shape[0]):
        t, j = (ids == e).nonzero(as_tuple=True)
        g, u = x[t] @ gate[e].t(), x[t] @ up[e].t()
        beyond += int((g > clamp).sum()) + int((u.abs() > clamp).sum())
        g, u = g.clamp_max(clamp), u.clamp(-clamp, clamp)
        out = out.index_add(0, t, w[t, j][:, None] * ((g * torch.sigmoid(g) * u) @ down[e].t()))
    return out, w, beyond


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("nt", [1, 40, 300])
def test_layer_runner_with_a_limit(cuda, dtype, nt):
    """a limit that holds back a third of the values, the shared expert's own limit beside it; bounds as test_layer_runner's.
    A value whose rounding crosses the limit has the gradient of the other side: eps / 2 of the values lie that near to it, so
    that the gradients' norms move by at most sqrt(eps) of themselves beside the roundings"""
    E, d, ff, k, clamp, sclamp = 16, 256, 136, 4, 0.5, 0.25
    g = gen(70 + nt)
    r = lambda *s, sc=1.0: torch.randn(*s, generator=g) * sc  # noqa: E731
    gate, up, down = (r(*s, sc=sc).to(dtype) for s, sc in (((E, ff, d), d ** -0.5), ((E, ff, d), d ** -0.5), ((E, d, ff), ff ** -0.5)))
    W_r, x, dy = r(E, d, sc=0.1), r(nt, d), r(nt, d, sc=0.1)
    on = lambda t: t.to(cuda)  # noqa: E731
    dev = mm16.Moe16Dev(on(gate), on(up), on(down), torch.arange(E, dtype=torch.int32, device=cuda), clamp)
    sh = mm16.Moe16Dev(on(gate[:1]), on(up[:1]), on(down[:1]), torch.zeros(1, dtype=torch.int32, device=cuda), sclamp)
    run = mm16.Moe16LayerRunner(dev, on(W_r), k, 300, shared=sh)
    out = run.forward(on(x)).clone()
    ids = run.ids[:nt * k].view(nt, k).long().cpu()
    leaves = [t.double().requires_grad_() for t in (x.to(dtype), gate, up, down)]
    want, w, beyond = _layer(leaves[0], W_r.double(), *leaves[1:], k, ids, clamp)
    assert beyond > 0.5 * nt * k * ff                            # of 2 nt k ff values
    xs = x.to(dtype).double()
    a, b = (xs @ gate[0].double().t()).clamp_max(sclamp), (xs @ up[0].double().t()).clamp(-sclamp, sclamp)
    S = (a * torch.sigmoid(a) * b) @ down[0].double().t()
    eps = torch.finfo(dtype).eps
    assert _rel(out, want.detach() + S) < 4 * eps
    assert _rel(run.forward(on(x), keep=True), want.detach() + S) < 4 * eps
    got = run.backward(on(dy))
    want.backward(dy.double())
    for name, t in (*zip(("dx", "gate", "up", "down"), leaves), ("dwts", w)):
        assert _rel(got[name], t.grad) < 8 * eps + math.sqrt(eps), name


def test_layer_runner_step_captured(cuda):
    """forward and backward in one graph, replayed on new inputs with eager work of another runner between"""
    def make(seed):
        g = gen(seed)
        r = lambda *s: (torch.randn(*s, generator=g) * 0.1).to(torch.bfloat16).to(cuda)  # noqa: E731
        E, d, ff, k, nt = 8, 64, 40, 2, 24
        dev = mm16.Moe16Dev(r(E, ff, d), r(E, ff, d), r(E, d, ff), torch.arange(E, dtype=torch.int32, device=cuda))
        x, dy = (torch.randn(3, nt, d, generator=g).to(cuda) for _ in range(2))
        return mm16.Moe16LayerRunner(dev, torch.randn(E, d, generator=g).to(cuda), k, nt), x, dy

    def step(run, x, dy):
        return {"out": run.forward(x, keep=True), **run.backward(dy)}
    (run, x, dy), (other, ox, ody) = make(1), make(2)
    want = [{n: t.clone() for n, t in step(run, x[i], dy[i]).items()} for i in range(3)]
    xin, dyin = x[0].clone(), dy[0].clone()
    st = torch.cuda.Stream()
    torch.cuda.synchronize()
    with torch.cuda.stream(st):
        step(run, xin, dyin)
    torch.cuda.synchronize()
    gr = torch.cuda.CUDAGraph()
    with torch.cuda.graph(gr, stream=st):
        out = step(run, xin, dyin)
    for i in (0, 1, 2, 1, 0):
        xin.copy_(x[i])
        dyin.copy_(dy[i])
        step(other, ox[i], ody[i])
        torch.cuda.synchronize()
        gr.replay()
        torch.cuda.synchronize()
        for n, t in out.items():
            assert torch.equal(t, want[i][n]), (i, n)
