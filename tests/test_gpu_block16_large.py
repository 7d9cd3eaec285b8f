"""Norms, their gradients, routing and adapters over more rows than a launch has blocks and more values than 32 bits count: the last
rows have the bits that a call of them alone gives, and the sums over all rows are exact on small integers."""
import pytest
import torch

from hyper_amd import mm16

pytestmark = pytest.mark.gpu
F32, BF = torch.float32, torch.bfloat16
LAST = 3000


def cuda_gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def test_norm_of_many_rows():
    m, n = (1 << 20) + 77, 4100
    assert m * n > 1 << 32
    x = torch.empty(m, n, dtype=BF, device="cuda").normal_(generator=cuda_gen(1))
    w = torch.rand(n, generator=cuda_gen(2), device="cuda")
    for kind in ("layer", "rms"):
        out, mean, rstd = torch.zeros_like(x), torch.zeros(m, device="cuda"), torch.zeros(m, device="cuda")
        mm16.norm(x, w, out, kind=kind, mean=mean, rstd=rstd)
        o, mu, r = torch.zeros(LAST, n, dtype=BF, device="cuda"), torch.zeros(LAST, device="cuda"), torch.zeros(LAST, device="cuda")
        mm16.norm(x[m - LAST:], w, o, kind=kind, mean=mu, rstd=r)
        assert torch.equal(out[m - LAST:], o) and torch.equal(mean[m - LAST:], mu) and torch.equal(rstd[m - LAST:], r)
        assert float(rstd.min()) > 0.5   # every row was normed (variances of 4100 normal values lie within a tenth of 1)


def test_norm_gradients_of_many_rows():
    """x of -2 .. 2, dy of -1 .. 1, rstd 1: every product and partial sum of dw is an integer far below 2^24"""
    m, n = (1 << 20) + 77, 4100
    x = torch.randint(-2, 3, (m, n), dtype=torch.int8, device="cuda", generator=cuda_gen(3))
    dy = torch.randint(-1, 2, (m, n), dtype=torch.int8, device="cuda", generator=cuda_gen(4))
    want = torch.zeros(n, dtype=torch.int64, device="cuda")
    for a in range(0, m, 1 << 16):
        want += (x[a:a + (1 << 16)] * dy[a:a + (1 << 16)]).sum(0, dtype=torch.int64)
    x, dy = x.to(BF), dy.to(BF)
    w, rstd, dx, dw = torch.rand(n, generator=cuda_gen(5), device="cuda"), torch.ones(m, device="cuda"), torch.zeros_like(x), torch.zeros(n, device="cuda")
    ws = torch.empty(mm16.norm_bwd_ws_bytes(m, n), dtype=torch.uint8, device="cuda")
    mm16.norm_bwd(x, dy, w, rstd, dx, kind="rms", dw=dw, ws=ws)
    assert torch.equal(dw.long(), want)
    d = torch.zeros(LAST, n, dtype=BF, device="cuda")
    mm16.norm_bwd(x[m - LAST:], dy[m - LAST:], w, rstd[m - LAST:], d, kind="rms")
    assert torch.equal(dx[m - LAST:], d)


def test_routing_of_many_tokens():
    nt, E, k = (1 << 23) + 100, 520, 4
    assert nt * E > 1 << 32
    logits = torch.empty(nt, E, device="cuda").normal_(generator=cuda_gen(6))
    how = dict(score="sigmoid", n_group=8, top_group=3, group_best=2)

    def route(l):
        ids, wts = torch.full((l.shape[0], k), -7, dtype=torch.int32, device="cuda"), torch.zeros(l.shape[0], k, device="cuda")
        mm16.route_groups(l, ids, wts, **how)
        return ids, wts
    ids, wts = route(logits)
    i, w = route(logits[nt - LAST:])
    assert torch.equal(ids[nt - LAST:], i) and torch.equal(wts[nt - LAST:], w)
    assert int(ids.min()) >= 0 and int(ids.max()) < E
    dl, d = torch.zeros(nt, E, dtype=BF, device="cuda"), torch.zeros(LAST, E, dtype=BF, device="cuda")
    mm16.route_groups_bwd(logits, ids, wts, dl, score="sigmoid")
    mm16.route_groups_bwd(logits[nt - LAST:], i, w, d, score="sigmoid")
    assert torch.equal(dl[nt - LAST:], d)


def test_adapters_of_many_rows():
    """small integers: exact whatever the tiles"""
    m, k, n, r = 620_000, 64, 7168, 8
    assert m * n > 1 << 32
    ints = lambda lo, hi, *s, seed: torch.randint(lo, hi + 1, s, dtype=torch.int8, device="cuda", generator=cuda_gen(seed)).to(BF)  # noqa: E731
    L = mm16.Lora16(ints(-1, 1, 5, r, k, seed=7), ints(-1, 1, 5, n, r, seed=8))
    x, out = ints(-1, 1, m, k, seed=9), ints(-2, 2, m, n, seed=10)
    ids = (torch.arange(m, device="cuda") // 1000 % 6 - 1).to(torch.int32)
    last = out[m - LAST:].clone()
    mm16.lora(L, x, ids, out, resid=out, ws=torch.empty(mm16.lora_ws_bytes(L, m), dtype=torch.uint8, device="cuda"))
    mm16.lora(L, x[m - LAST:], ids[m - LAST:].contiguous(), last, resid=last, ws=torch.empty(mm16.lora_ws_bytes(L, LAST), dtype=torch.uint8, device="cuda"))
    assert torch.equal(out[m - LAST:], last)
