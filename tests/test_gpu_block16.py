"""A layer with its norm and its router, forward and backward, against 64-bit autograd, and the operators as they follow each other.

Bounds are relative norms, in steps eps of the 16-bit type, each rounding half a step and independent of the others: the output
4 eps and the routing weights' gradient 8 eps as for the layer without them; the logits' gradient w (dw - sum w dw) carries the
latter twice and half a step of its own (16.5 eps), the router's weights and its part of the rows half a step more (17 eps); the
norm's backward pass takes two of d directions out of the rows and adds fp32 arithmetic (20 eps covers 17 by the 2 / d = 1 % of it)."""
import pytest
import torch

from hyper_amd import mm16
from tests.helpers import gen
from tests.test_gpu_route_groups import route64

pytestmark = pytest.mark.gpu
TYPES = [torch.bfloat16, torch.float16]


def rel(a, b):
    return float((a.double().cpu() - b).norm() / b.norm())


def norm64(x, w, b, kind, eps):
    mean = x.mean(1, keepdim=True) if kind == "layer" else 0.0
    y = (x - mean) / (((x - mean) ** 2).mean(1, keepdim=True) + eps).sqrt() * w
    return y if b is None else y + b


def layer64(x, nw, nb, W_r, gate, up, down, ids, kind, score, renorm, scale):
    """the layer for given experts, differentiable: (output, weights)"""
    xn = norm64(x, nw, nb, kind, 1e-5)
    l = xn @ W_r.t()
    on, at = ids >= 0, ids.clamp_min(0)
    s = (torch.softmax(l, 1) if score == "softmax" else torch.sigmoid(l)).gather(1, at)
    s = torch.where(on, s, torch.zeros_like(s))
    w = s / s.sum(1, keepdim=True) * scale if renorm else s * scale
    out = torch.zeros_like(x)
    for e in range(gate.shape[0]):
        t, j = (ids == e).nonzero(as_tuple=True)
        g, u = xn[t] @ gate[e].t(), xn[t] @ up[e].t()
        out = out.index_add(0, t, w[t, j][:, None] * ((g * torch.sigmoid(g) * u) @ down[e].t()))
    return out, w


def make(dtype, kind, score, renorm, w_type, dev, max_rows, seed, masked=False):
    E, d, ff, k = 16, 256, 136, 4
    g = gen(seed)
    r = lambda *s, sc=1.0: torch.randn(*s, generator=g) * sc  # noqa: E731
    gate, up, down = (r(*s, sc=sc).to(dtype) for s, sc in (((E, ff, d), d ** -0.5), ((E, ff, d), d ** -0.5), ((E, d, ff), ff ** -0.5)))
    W_r, nw, nb = r(E, d, sc=0.1).to(w_type), 1 + r(d, sc=0.2), r(d, sc=0.1) if kind == "layer" else None
    bias = r(E, sc=0.05)
    if masked:
        bias[::3] = -float("inf")
    on = lambda t: None if t is None else t.to(dev)  # noqa: E731
    how = dict(score=score, n_group=4, top_group=2, group_best=2, renorm=renorm, scale=1.5)
    run = mm16.Moe16LayerRunner(mm16.Moe16Dev(on(gate), on(up), on(down), torch.arange(E, dtype=torch.int32, device=dev)), on(W_r), k, max_rows,
                                norm=mm16.Norm16(on(nw), on(nb), 1e-5, kind), router=mm16.Router16(bias=on(bias), **how))
    return run, (nw, nb, W_r, gate, up, down), dict(how, bias=bias), g


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("kind,score,renorm,w_type", [("rms", "sigmoid", True, torch.float32), ("layer", "softmax", True, torch.bfloat16),
                                                      ("rms", "softmax", False, torch.float32), ("layer", "sigmoid", False, torch.bfloat16)])
@pytest.mark.parametrize("nt", [1, 2, 5, 40, 300])
def test_layer_with_norm_and_router(dtype, kind, score, renorm, w_type, nt):
    dev = torch.device("cuda:0")
    run, params, how, g = make(dtype, kind, score, renorm, w_type, dev, 300, 7 * nt + 1, masked=nt == 40)
    x, dy, add, by = torch.randn(nt, 256, generator=g) + 0.3, *(torch.randn(nt, 256, generator=g) * 0.1 for _ in range(3))
    eps = torch.finfo(dtype).eps
    out = run.forward(x.to(dev)).clone()
    ids, wts = run.ids[:4 * nt].view(nt, 4).cpu(), run.wts[:4 * nt].view(nt, 4)
    assert torch.equal(ids, route64(run.logits[:nt].cpu(), 4, **how)[0])   # the routing of the logits as they are
    # the reference's leaves; the experts see the normed rows rounded to 16 bits, the router's product the unrounded ones
    leaves = [None if t is None else t.double().requires_grad_() for t in (x, *params)]
    want, w = layer64(*leaves, ids.long(), kind, score, renorm, 1.5)
    w.retain_grad()
    assert rel(out, want.detach()) < 4 * eps
    assert rel(wts, w.detach()) < 1e-4 if nt > 5 else True   # fp32 logits
    assert rel(run.forward(x.to(dev), keep=True), want.detach()) < 4 * eps
    got = run.backward(dy.to(dev))
    want.backward(dy.double())
    assert rel(got["dwts"], w.grad) < 8 * eps
    for name, t in zip(("dx", "norm_w", "norm_b", "W_r", "gate", "up", "down"), leaves):
        if t is None:
            assert got[name] is None
        else:
            assert rel(got[name], t.grad) < (8 if name in ("gate", "up", "down") else 20) * eps, name
    # what backward leaves out comes in at the rows that the experts see, and the residual stream's gradient at the end
    more = run.backward(dy.to(dev), dx_add=add.to(dev), resid=by.to(dev))
    xg = x.double().requires_grad_()
    norm64(xg, *(None if t is None else t.double() for t in params[:2]), kind, 1e-5).backward(add.double())
    assert rel(more["dx"] - got["dx"], xg.grad + by.double()) < 1e-4
    for name in ("gate", "up", "down", "W_r", "dwts"):
        assert torch.equal(more[name], got[name]), name


def test_the_reference_gradients_are_differences():
    """the 64-bit layer that the gradients are compared with: central differences along each leaf's gradient say its square"""
    g = gen(1)
    E, d, ff, k, nt = 8, 32, 24, 3, 6
    r = lambda *s: torch.randn(*s, generator=g, dtype=torch.float64)  # noqa: E731
    leaves = [r(nt, d), 1 + 0.1 * r(d), 0.1 * r(d), 0.3 * r(E, d), *(d ** -0.5 * r(E, a, b) for a, b in ((ff, d), (ff, d), (d, ff)))]
    ids, dy = torch.stack([torch.randperm(E, generator=g)[:k] for _ in range(nt)]), r(nt, d)
    for kind, score, renorm in (("layer", "sigmoid", True), ("layer", "softmax", False), ("rms", "softmax", True)):
        x = [t.clone().requires_grad_() for t in leaves]
        (layer64(*x, ids, kind, score, renorm, 1.5)[0] * dy).sum().backward()
        for i, t in enumerate(x):
            step = 1e-5 / float(t.grad.norm())
            hi, lo = ((layer64(*[a + s * step * t.grad if j == i else a for j, a in enumerate(leaves)], ids, kind, score, renorm, 1.5)[0] * dy).sum() for s in (1, -1))
            assert abs(float((hi - lo) / (2 * step)) / float((t.grad ** 2).sum()) - 1) < 1e-5, (kind, i)


def test_tokens_without_experts():
    """every expert masked by the selection bias: no output, no gradient but the residual's, and finite everywhere"""
    dev = torch.device("cuda:0")
    run, _, _, g = make(torch.bfloat16, "rms", "sigmoid", True, torch.float32, dev, 20, 3)
    run.router.how["bias"].fill_(-float("inf"))
    x, dy = torch.randn(20, 256, generator=g).to(dev), torch.randn(20, 256, generator=g).to(dev)
    for n in (1, 20):   # by ids and grouped
        assert (run.forward(x[:n]) == 0).all() and (run.ids[:4 * n] == -1).all() and (run.wts[:4 * n] == 0).all()
    assert (run.forward(x, keep=True) == 0).all()
    got = run.backward(dy, resid=dy)
    assert torch.equal(got["dx"], dy)
    for name in ("W_r", "norm_w", "gate", "up", "down", "dwts"):
        assert (got[name] == 0).all(), name


def test_layer_of_no_rows():
    dev = torch.device("cuda:0")
    run, _, _, _ = make(torch.float16, "layer", "sigmoid", True, torch.float32, dev, 4, 5)
    none = torch.empty(0, 256, device=dev)
    assert run.forward(none, keep=True).shape == (0, 256)
    got = run.backward(none)
    assert got["dx"].shape == (0, 256)
    for name in ("W_r", "norm_w", "norm_b", "gate", "up", "down"):
        assert (got[name] == 0).all(), name


def test_layer_step_captured_and_replayed():
    dev = torch.device("cuda:0")
    run, _, _, _ = make(torch.bfloat16, "layer", "sigmoid", True, torch.float32, dev, 50, 9)
    x, dy = torch.empty(50, 256, device=dev), torch.empty(50, 256, device=dev)

    def step():
        out = run.forward(x, keep=True)
        return {"out": out, **run.backward(dy, resid=dy)}

    def fill(seed):
        x.copy_(torch.randn(50, 256, generator=gen(seed)))
        dy.copy_(torch.randn(50, 256, generator=gen(seed + 1)))
    fill(1)
    st = torch.cuda.Stream()
    with torch.cuda.stream(st):
        step()
    torch.cuda.synchronize()
    gr = torch.cuda.CUDAGraph()
    with torch.cuda.graph(gr, stream=st):
        captured = step()
    for seed in range(3):
        fill(10 * seed + 20)
        eager = {n: t.clone() for n, t in step().items()}
        torch.cuda.synchronize()
        for t in captured.values():
            t.zero_()
        gr.replay()
        torch.cuda.synchronize()
        for n, t in eager.items():
            assert torch.equal(captured[n], t), (seed, n)


def test_runner_refusals():
    dev = torch.device("cuda:0")
    E, d = 8, 64
    m = mm16.Moe16Dev(*(torch.zeros(*s, dtype=torch.bfloat16, device=dev) for s in ((E, 40, d), (E, 40, d), (E, d, 40))), torch.arange(E, dtype=torch.int32, device=dev))
    W_r, w = torch.zeros(E, d, device=dev), torch.ones(d, device=dev)
    with pytest.raises(ValueError, match="64 weights"):
        mm16.Moe16LayerRunner(m, W_r, 2, 4, norm=mm16.Norm16(w[:32].contiguous()))
    with pytest.raises(ValueError, match="bias must hold"):
        mm16.Moe16LayerRunner(m, W_r, 2, 4, router=mm16.Router16(bias=w[:4].contiguous()))
    with pytest.raises(ValueError, match="no b"):
        mm16.Norm16(w, w)
    with pytest.raises(ValueError, match="unknown norm"):
        mm16.Norm16(w, kind="group")
    with pytest.raises(ValueError, match="unknown score"):
        mm16.Router16("tanh")
    run = mm16.Moe16LayerRunner(m, W_r, 2, 4, router=mm16.Router16())
    x = torch.ones(4, d, device=dev)
    run.forward(x, keep=True)
    with pytest.raises(ValueError, match="goes with a norm"):
        run.backward(x, resid=x)
    with pytest.raises(ValueError, match="dx_add"):
        run.backward(x, dx_add=x[:2])


def test_adapters_beside_a_norm_and_a_projection():
    """a serving step: norm, projection, every request's adapter into it -- the composition of the three formulas"""
    dev = torch.device("cuda:0")
    g = gen(4)
    for m, how in ((9, "each"), (400, "runs")):
        d, n, r = 512, 384, 16
        dt = torch.bfloat16
        x, w = torch.randn(m, d, generator=g), 1 + 0.1 * torch.randn(d, generator=g)
        W, A, B = ((torch.randn(*s, generator=g) * s[-1] ** -0.5).to(dt) for s in ((n, d), (5, r, d), (5, n, r)))
        ids = torch.randint(-1, 5, (m,), generator=g).to(torch.int32) if how == "each" else torch.arange(m).mul(6).div(m, rounding_mode="floor").sub(1).to(torch.int32)
        y, out = torch.empty(m, d, dtype=dt, device=dev), torch.empty(m, n, device=dev)
        L = mm16.Lora16(A.to(dev), B.to(dev))
        mm16.norm(x.to(dev), w.to(dev), y, kind="rms")
        mm16.linear(W.to(dev), y, out)
        mm16.lora(L, y, ids.to(dev), out, resid=out, ws=torch.empty(mm16.lora_ws_bytes(L, m), dtype=torch.uint8, device=dev))
        yn = norm64(x.double(), w.double(), None, "rms", 1e-5)
        want = yn @ W.double().t()
        for t, a in enumerate(ids.tolist()):
            if a >= 0:
                want[t] += B[a].double() @ (A[a].double() @ yn[t])
        assert rel(out, want) < 2 * torch.finfo(dt).eps   # the normed rows' half steps, in both products
