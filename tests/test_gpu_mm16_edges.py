"""The 16-bit products at the ends of their ranges: many pairs, infinities and NaN, slot tables that change, empty calls.

Products are on small integers, exact in any order of fp32 sums, as in test_gpu_mm16."""
import pytest
import torch

from hyper_amd import mm16

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
