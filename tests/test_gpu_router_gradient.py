"""The router of a layer: its weights forward, by ids and grouped, and its own gradients, each apart from the experts'.

From the routing weights' gradient dwts as backward returns it, the logits' gradient dl is known in 64 bits.  With v = 2^-16, what two
bfloat16 values leave of a number (each half a step, 2^-8 of what it rounds), and U = 2^-23 a unit in the last place of a float32 sum's term:
  dW_r = dl^T x    of the rows as the experts see them (16 bits):  (3 v + (4 nt + 16) U) |dl|^T |x|
  dx += dl W_r     the share alone is the difference of dx with and without it:  (3 v + (4 E + 16) U) |dl| |W_r| + 4 U |dx|
dl itself is kept within 2^-24 and what 64 bits leave of its terms (w |dwts| scale, 1e-12)."""
import pytest
import torch

from hyper_amd import mm16
from tests.helpers import gen
from tests.test_gpu_mm16 import within
from tests.test_gpu_route_groups import route64

pytestmark = pytest.mark.gpu
BF, FP, F32 = torch.bfloat16, torch.float16, torch.float32
v, U = 2.0 ** -16, 2.0 ** -23
HOW = [("sigmoid", True), ("softmax", True), ("softmax", False), ("sigmoid", False)]


def make(dtype, w_type, score, renorm, E, k, d, max_rows, dev, seed, norm=False):
    g = gen(seed)
    ff = 72
    r = lambda *s, sc: torch.randn(*s, generator=g) * sc  # noqa: E731
    dev_ = mm16.Moe16Dev(*(r(*s, sc=s[-1] ** -0.5).to(dtype).to(dev) for s in ((E, ff, d), (E, ff, d), (E, d, ff))),
                         torch.arange(E, dtype=torch.int32, device=dev))
    W_r, nw = r(E, d, sc=2 * d ** -0.5).to(w_type).to(dev), 1 + r(d, sc=0.2).to(dev)
    how = dict(score=score, n_group=4, top_group=3, group_best=2, renorm=renorm, scale=1.5)
    run = mm16.Moe16LayerRunner(dev_, W_r, k, max_rows, norm=mm16.Norm16(nw) if norm else None, router=mm16.Router16(**how))
    return run, how, g


def logits_grad64(l, ids, dwts, score, renorm, scale):
    l = l.double().cpu().requires_grad_()
    s = (torch.softmax(l, 1) if score == "softmax" else torch.sigmoid(l)).gather(1, ids)
    w = s / s.sum(1, keepdim=True) * scale if renorm else s * scale
    (w * dwts.double().cpu()).sum().backward()
    terms = (w.detach().abs() * dwts.double().cpu().abs()).sum(1, keepdim=True)   # what dl's terms cancel from
    return l.grad, terms


@pytest.mark.parametrize("dtype", [BF, FP])
@pytest.mark.parametrize("w_type", [F32, BF])
@pytest.mark.parametrize("score,renorm", HOW)
@pytest.mark.parametrize("nt,E,size", [(1, 16, 0.1), (40, 16, 0.1), (300, 60, 0.1), (64, 128, 1e-4), (33, 60, 2e-5)])
def test_router_gradients_alone(dtype, w_type, score, renorm, nt, E, size):
    """size: of dy.  Small ones give logits' gradients far below what fp16 holds"""
    dev = torch.device("cuda:0")
    d, k = 192, 4
    run, how, g = make(dtype, w_type, score, renorm, E, k, d, 300, dev, nt + E)
    x, dy = torch.randn(nt, d, generator=g).to(dev), (size * torch.randn(nt, d, generator=g)).to(dev)
    run.forward(x, keep=True)
    ids = run.ids[:nt * k].view(nt, k).long().cpu()
    got = run.backward(dy)
    router, run.router = run.router, None
    without = run.backward(dy)["dx"]
    run.router = router
    assert float(got["dwts"].abs().max()) > 0
    dl, terms = logits_grad64(run.logits[:nt], ids, got["dwts"], score, renorm, 1.5)
    dl_err = 2.0 ** -24 * dl.abs() + 1e-12 * terms
    x16, W = run.x16[:nt].double().cpu(), run.W_r.double().cpu()
    within(got["W_r"], dl.t() @ x16, (3 * v + (4 * nt + 16) * U) * (dl.abs().t() @ x16.abs()) + dl_err.t() @ x16.abs(), "W_r")
    share = got["dx"].double().cpu() - without.double().cpu()
    bound = (3 * v + (4 * E + 16) * U) * (dl.abs() @ W.abs()) + dl_err @ W.abs() + 4 * U * got["dx"].double().cpu().abs()
    off = (share - dl @ W).abs()
    assert (off <= bound).all(), (float((off / bound).max()), float(off.max()))


@pytest.mark.parametrize("w_type", [F32, BF])
@pytest.mark.parametrize("nt", [1, 2, 3, 5, 40])
def test_routing_weights_at_every_number_of_rows(w_type, nt):
    """by ids (up to two rows) and grouped: the logits within a float32 product's bound, the weights those of the logits"""
    dev = torch.device("cuda:0")
    d, E, k = 192, 60, 4
    for i, (score, renorm) in enumerate(HOW):
        run, how, g = make((BF, FP)[i % 2], w_type, score, renorm, E, k, d, 40, dev, 10 * nt + i)
        x = torch.randn(nt, d, generator=g)
        run.forward(x.to(dev))
        W = run.W_r.double().cpu()
        logits = run.logits[:nt].cpu()
        within(logits, x.double() @ W.t(), (d + 4) * U * (x.double().abs() @ W.abs().t()), "logits")
        ids, w = route64(logits, k, **how)
        assert torch.equal(run.ids[:nt * k].view(nt, k).cpu(), ids)
        within(run.wts[:nt * k].view(nt, k), w, 1e-12 * w.abs() + 1e-30, "weights")


def test_router_gradient_of_no_rows():
    dev = torch.device("cuda:0")
    for dtype in (BF, FP):
        for w_type in (F32, BF):
            run, _, _ = make(dtype, w_type, "sigmoid", True, 60, 4, 192, 8, dev, 3)
            none = torch.empty(0, 192, device=dev)
            run.forward(none, keep=True)
            got = run.backward(none)
            assert got["dx"].shape == (0, 192) and got["W_r"].shape == (60, 192) and (got["W_r"] == 0).all()


@pytest.mark.parametrize("dtype,w_type", [(BF, F32), (FP, F32), (FP, BF)])
def test_router_step_captured_and_replayed(dtype, w_type):
    """many rows (the norm's gradient by blocks and their join): the eager bits, replay after replay"""
    dev = torch.device("cuda:0")
    nt, E, d = 1100, 60, 256
    run, _, _ = make(dtype, w_type, "sigmoid", True, E, 4, d, nt, dev, 9, norm=True)
    x, dy = torch.empty(nt, d, device=dev), torch.empty(nt, d, device=dev)

    def step():
        out = run.forward(x, keep=True)
        return {"out": out, **{n: t for n, t in run.backward(dy, resid=dy).items() if t is not None}}

    def fill(seed):
        x.copy_(torch.randn(nt, d, generator=gen(seed)))
        dy.copy_(torch.randn(nt, d, generator=gen(seed + 1)))
    fill(1)
    st = torch.cuda.Stream()
    with torch.cuda.stream(st):
        step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=st):
        captured = step()
    for seed in range(3):
        fill(10 * seed + 20)
        eager = {n: t.clone() for n, t in step().items()}
        torch.cuda.synchronize()
        for t in captured.values():
            t.zero_()
        graph.replay()
        torch.cuda.synchronize()
        for n, t in eager.items():
            assert torch.equal(captured[n], t), (seed, n)
