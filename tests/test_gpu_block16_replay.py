"""Norms, their gradients and adapters at the sizes whose kernels differ, captured into a graph, replayed, and on another stream: the
eager bits every time.  (The calls of few rows and routing have such tests beside their own.)"""
import pytest
import torch

from hyper_amd import mm16
from tests.helpers import gen

pytestmark = pytest.mark.gpu
F32, BF, FP = torch.float32, torch.bfloat16, torch.float16


def replay(fill, step, buffers):
    """step(outputs, stream): eager, captured and on a stream of its own, each with outputs of its own, over new inputs"""
    a, b, c = buffers(), buffers(), buffers()
    fill(0)
    step(b, None)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step(b, None)
    for seed in range(1, 4):
        fill(seed)
        step(a, None)
        torch.cuda.synchronize()
        for t in b.values():
            t.fill_(7)
        graph.replay()
        torch.cuda.synchronize()
        s = torch.cuda.Stream()
        step(c, s)
        s.synchronize()
        for name in a:
            assert torch.equal(a[name], b[name]) and torch.equal(a[name], c[name]), (seed, name)
            assert not a[name].isnan().any()


# blocks that take several rows' turns, with the join; rows between the powers of two; odd rows; several pieces a thread; rows longer than the registers
@pytest.mark.parametrize("m,n,xt,kind", [(2100, 512, F32, "layer"), (2100, 1200, BF, "rms"), (1100, 2048, FP, "layer"), (600, 6001, F32, "rms"),
                                         (400, 9001, BF, "layer"), (300, 14000, F32, "layer"), (37, 20000, F32, "layer"), (37, 20001, BF, "rms")])
def test_norms_and_gradients(m, n, xt, kind):
    dev = torch.device("cuda:0")
    x, d, dy, w = torch.empty(m, n, dtype=xt, device=dev), torch.empty(m, n, dtype=xt, device=dev), torch.empty(m, n, dtype=BF, device=dev), torch.rand(n, device=dev)
    ws = torch.empty(mm16.norm_bwd_ws_bytes(m, n), dtype=torch.uint8, device=dev)
    layer = kind == "layer"

    def fill(seed):
        g = gen(100 * seed + n)
        for t in (x, d, dy):
            t.copy_(torch.randn(m, n, generator=g).to(t.dtype))

    def buffers():
        o = dict(y=torch.empty(m, n, device=dev, dtype=BF), total=torch.empty_like(x), rstd=torch.empty(m, device=dev), dx=torch.empty_like(x),
                 dw=torch.empty(n, device=dev))
        return {**o, "mean": torch.empty(m, device=dev), "db": torch.empty(n, device=dev)} if layer else o

    def step(o, stream):
        mm16.norm(x, w, o["y"], b=w if layer else None, kind=kind, add=d, total=o["total"], mean=o.get("mean"), rstd=o["rstd"], stream=stream)
        mm16.norm_bwd(o["total"], dy, w, o["rstd"], o["dx"], mean=o.get("mean"), kind=kind, resid=d, dw=o["dw"], db=o.get("db"), ws=ws, stream=stream)
    replay(fill, step, buffers)


# tall tiles and tiles of 16 rows; each number of ranks; with and without a residual, odd outputs, both output types
@pytest.mark.parametrize("m,k,n,r,ot,resid", [(700, 520, 384, 16, BF, True), (700, 520, 384, 64, F32, True), (700, 256, 392, 64, BF, False), (300, 264, 257, 40, BF, True),
                                              (300, 520, 264, 128, BF, True), (300, 264, 264, 256, F32, True), (24, 2048, 264, 64, BF, True), (24, 512, 65, 200, F32, False)])
def test_adapters(m, k, n, r, ot, resid):
    dev = torch.device("cuda:0")
    g = gen(m + r)
    L = mm16.Lora16((torch.randn(5, r, k, generator=g) * k ** -0.5).to(BF).to(dev), (torch.randn(5, n, r, generator=g) * r ** -0.5).to(BF).to(dev), torch.rand(5, generator=g).to(dev))
    x, base, ids = torch.empty(m, k, dtype=BF, device=dev), torch.empty(m, n, dtype=ot, device=dev), torch.empty(m, dtype=torch.int32, device=dev)
    ws = torch.empty(mm16.lora_ws_bytes(L, m), dtype=torch.uint8, device=dev)

    def fill(seed):
        g = gen(100 * seed + m)
        x.copy_(torch.randn(m, k, generator=g).to(BF))
        base.copy_(torch.randn(m, n, generator=g).to(ot))
        runs = torch.sort(torch.randint(0, m, (4,), generator=g)).values
        ids.copy_(torch.randint(-1, 5, (5,), generator=g)[torch.bucketize(torch.arange(m), runs, right=True)].to(torch.int32))

    def step(o, stream):
        mm16.lora(L, x, ids, o["out"], resid=base if resid else None, ws=ws, stream=stream)
    replay(fill, step, lambda: dict(out=torch.empty(m, n, dtype=ot, device=dev)))
