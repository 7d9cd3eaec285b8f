"""16-bit calls of more rows, columns or pairs than one direction of a launch holds (2^32 threads, beyond which it runs the rest
of the division and reports nothing): taken, or refused by name."""
import ctypes

import pytest
import torch

import hyper_amd
from hyper_amd import lib, mm16
from tests.test_mm16_args import BF16, P, _dev

S = hyper_amd.HY_EBAD_SHAPE
BIG = 1 << 30


def test_too_many_tiles_are_refused():
    L, odd = lib(), ctypes.c_void_p(66)
    for at in (P, odd):                                        # the tile kernels, and the one for any alignment
        assert L.hy_linear(BF16, P, 8, BIG, 8, at, 8, 8192, None, 0, None, 0, None, 0, P, BF16, BIG, None) == S
        assert b"tiles" in L.hy_last_error()
        assert L.hy_linear_glu(BF16, P, P, 8, BIG, 8, at, 8, 8192, 0.0, None, None, P, BIG, None) == S
        assert L.hy_linear_dx(BF16, P, BIG, 8, BIG, at, 8, 8192, None, 0, P, BF16, BIG, None) == S
        assert L.hy_linear_dw(BF16, at, BIG, P, 8192, 8, BIG, 8192, P, BF16, 8192, None, 0, None, 0, None) == S
    m = _dev(ff=BIG, n=8, E=2)
    assert L.hy_moe16_gate_up(ctypes.byref(m), P, 8, 2, None, 4096, P, P, P, 1024, None, None, P, None) == S
    assert L.hy_moe16_dw(ctypes.byref(m), BF16, P, BIG, 1, BIG, P, 8192, 1, 8192, 64, P, P, P, 2, P, BF16, 0, None) == S


def test_more_tokens_than_a_launch_holds_are_refused():
    L = lib()
    for fn in (L.hy_moe_reduce, L.hy_moe_reduce_residual):
        assert fn(None, None, P, 2, P, 64, 1 << 24, P, None) == S and b"tokens" in L.hy_last_error()
    b = lambda *s: torch.zeros(*s, dtype=torch.bfloat16)  # noqa: E731
    for E, rows in ((2, 1 << 23), (1024, 1 << 21), (17, (1 << 26) - 8)):
        m = mm16.Moe16Dev(b(1, 8, 4), b(1, 8, 4), b(1, 4, 8), torch.zeros(E, dtype=torch.int32))
        with pytest.raises(ValueError, match="one launch"):
            mm16.Moe16LayerRunner(m, torch.zeros(E, 4), 1, rows)


def _rows(dev, n, w, seed):
    """n rows of w small integers that depend on the row's number, made without more memory than they take"""
    r = torch.arange(n, device=dev, dtype=torch.int32)[:, None]
    return torch.remainder(r * (2 * torch.arange(w, device=dev, dtype=torch.int32) + seed) + (r >> 9), 7).sub_(3).to(torch.bfloat16)


@pytest.mark.gpu
@pytest.mark.parametrize("w", [8, 7])
def test_one_row_of_many_columns(cuda, w):
    n = (1 << 27) + 9
    W = _rows(cuda, n, w, 3)
    x = torch.arange(w, device=cuda).sub(2).to(torch.bfloat16)[None]
    out = torch.full((1, n), 77.0, dtype=torch.bfloat16, device=cuda)
    mm16.linear(W, x, out)
    # (sums of eight integers; in pieces, since library products of so many rows leave their end out as well)
    bad = sum(int((out[0, at:at + (1 << 22)] != (W[at:at + (1 << 22)].float() * x[0].float()).sum(1).to(torch.bfloat16)).sum()) for at in range(0, n, 1 << 22))
    assert bad == 0
    h, g, u = (torch.full((1, n), 77.0, dtype=torch.bfloat16, device=cuda) for _ in range(3))
    mm16.linear_glu(W, W, x, h, g=g, u=u)
    bad = int((g != out).sum()) + int((u != out).sum()) + int((h == 77.0).sum())
    assert bad == 0


@pytest.mark.gpu
@pytest.mark.parametrize("ff", [2, 8])
def test_activation_gradient_of_many_pairs(cuda, ff):
    n = (1 << 26) + 5
    g, u, dh = (_rows(cuda, n, ff, s) for s in (1, 5, 9))
    dg, du, hw = (torch.full((n, ff), 77.0, dtype=torch.bfloat16, device=cuda) for _ in range(3))
    dw = torch.full((n,), 77.0, device=cuda)
    mm16.swiglu_bwd(g, u, dh, None, dg, du, hw, dw)
    left = int((dw == 77.0).sum()) + sum(int((t == 77.0).sum()) for t in (dg, du, hw))
    assert left == 0
    # the last rows (and rows around the first grid row's end) as a call of their own
    for at in (0, (1 << 24) - 8, n - 37):
        r = slice(at, at + 37)
        few = [torch.empty(37, ff, dtype=torch.bfloat16, device=cuda) for _ in range(3)] + [torch.empty(37, device=cuda)]
        mm16.swiglu_bwd(g[r].clone(), u[r].clone(), dh[r].clone(), None, *few)
        assert all(torch.equal(a[r], b) for a, b in zip((dg, du, hw, dw), few))


@pytest.mark.gpu
def test_combine_of_many_tokens(cuda):
    nt, n = (1 << 24) + 3, 4
    y = _rows(cuda, nt, n, 3).float()
    ids = torch.arange(nt, dtype=torch.int32, device=cuda) % 3
    b = torch.zeros(2, 8, n, dtype=torch.bfloat16, device=cuda)
    m = mm16.Moe16Dev(b, b, None, torch.tensor([0, -1, 1], dtype=torch.int32, device=cuda))
    out = torch.full((nt, n), 77.0, device=cuda)
    mm16.moe16_reduce(m, None, None, y, 1, out, nt, ids)
    y[ids == 1] = 0
    bad = int((out != y).sum())
    assert bad == 0
