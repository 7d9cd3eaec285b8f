"""Outputs of the norms and of the routing gradient in the place of other matrices: what a row's kernel could overwrite before it is
read, and two outputs in one place, are refused before any device work; what is allowed gives the bits of places of their own."""
import ctypes

import pytest
import torch

import hyper_amd
from hyper_amd import lib, mm16
from tests.helpers import gen
from tests.test_block16_args import BF16, F16, F32, P, S, _norm

Q = ctypes.c_void_p(1 << 16)
R = ctypes.c_void_p(1 << 17)


def test_norm_outputs_in_the_place_of_add():
    """other strides or another type's size"""
    message = lambda: lib().hy_last_error()  # noqa: E731
    assert _norm(add=Q, lda=64, out=Q, ot=BF16) == S and b"out takes the place of add" in message()
    assert _norm(add=Q, lda=64, out=Q, ot=F32, ldo=72) == S and _norm(add=Q, lda=0, out=Q, ot=F32) == S
    assert _norm(xt=BF16, add=Q, lda=64, out=R, out32=Q, ld32=64) == S and b"out32 takes the place of add" in message()
    assert _norm(add=Q, lda=96, out=R, out32=Q, ld32=64) == S
    assert _norm(add=Q, lda=64, out=Q, ot=BF16, m=1) == S


def test_norm_outputs_in_one_place():
    message = lambda: lib().hy_last_error()  # noqa: E731
    assert _norm(total=Q, ldt=64, out=Q, ot=F32) == S and b"total and out are one place" in message()
    assert _norm(total=Q, ldt=64, out=Q, ot=BF16) == S and _norm(total=Q, ldt=64, out=R, out32=Q, ld32=64) == S
    assert _norm(out=Q, ot=F32, out32=Q, ld32=64) == S and b"out and out32 are one place" in message()
    assert _norm(x=P, total=P, ldt=64, out=P, ot=F32) == S   # both in x's place


def test_logits_gradient_in_the_place_of_the_logits():
    def call(dl=P, ty=F32, ldd=64, ls=64, nt=3):
        return lib().hy_moe_route_groups_bwd(P, ls, 64, 1, Q, 6, 1, 1.0, R, dl, ty, ldd, nt, None)
    assert call(ty=BF16) == S and b"dlogits takes the place of logits" in lib().hy_last_error()
    assert call(ty=F16) == S and call(ldd=72) == S and call(ls=80) == S and call(ty=BF16, nt=1) == S


@pytest.mark.gpu
@pytest.mark.parametrize("n", [7, 512, 1001, 4096, 9001, 20000])
def test_norm_in_the_place_of_add(n):
    dev = torch.device("cuda:0")
    g = gen(n)
    for dt in (torch.float32, torch.bfloat16):
        x, d = (torch.randn(40, n, generator=g).to(dt).to(dev) for _ in range(2))
        w = torch.rand(n, generator=g).to(dev)
        for kind in ("layer", "rms"):
            total, out = torch.empty_like(x), torch.empty_like(x)
            mm16.norm(x, w, out, kind=kind, add=d, total=total)
            a, t = d.clone(), torch.empty_like(x)
            mm16.norm(x, w, a, kind=kind, add=a, total=t)
            assert torch.equal(a, out) and torch.equal(t, total), (n, dt, kind)
            if dt is torch.float32:
                a = d.clone()
                mm16.norm(x, w, None, kind=kind, add=a, total=t, out32=a)
                assert torch.equal(a, out) and torch.equal(t, total), (n, kind)


@pytest.mark.gpu
@pytest.mark.parametrize("E", [5, 64, 100, 256, 1000])
def test_logits_gradient_takes_the_place_of_the_logits(E):
    dev = torch.device("cuda:0")
    g = gen(E)
    nt, k = 37, 4
    logits = torch.randn(nt, E + 3, generator=g).to(dev)[:, :E]
    ids = torch.stack([torch.randperm(E, generator=g)[:k] for _ in range(nt)]).to(torch.int32).to(dev)
    dwts = torch.randn(nt, k, generator=g).to(dev)
    for score in ("softmax", "sigmoid"):
        for renorm in (True, False):
            want = torch.empty(nt, E, device=dev)
            mm16.route_groups_bwd(logits, ids, dwts, want, score=score, renorm=renorm)
            wide = logits._base.clone()
            mm16.route_groups_bwd(wide[:, :E], ids, dwts, wide[:, :E], score=score, renorm=renorm)
            assert torch.equal(wide[:, :E], want) and torch.equal(wide[:, E:], logits._base[:, E:]), (E, score, renorm)
