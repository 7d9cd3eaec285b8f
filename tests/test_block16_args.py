"""Argument checks of the norms, of routing with groups and of the low-rank adapters, which come before any device work: codes
and messages of the C entries, and the Python wrappers' ValueErrors."""
import ctypes

import pytest
import torch

import hyper_amd
from hyper_amd import lib, mm16

I, S, U, OK = hyper_amd.HY_EINVAL, hyper_amd.HY_EBAD_SHAPE, hyper_amd.HY_EUNSUPPORTED_TYPE, hyper_amd.HY_OK
P = ctypes.c_void_p(64)
ODD = ctypes.c_void_p(65)
TWO = ctypes.c_void_p(66)
BF16, F16, F32 = 30, 1, 0


def _norm(kind=0, xt=F32, x=P, ldx=64, add=None, lda=0, total=None, ldt=0, w=P, b=P, eps=1e-5, m=8, n=64, out=P, ot=BF16, ldo=64, out32=None, ld32=0,
          mean=None, rstd=None):
    return lib().hy_norm(kind, xt, x, ldx, add, lda, total, ldt, w, b, eps, m, n, out, ot, ldo, out32, ld32, mean, rstd, None)


def test_norm_refusals():
    assert _norm(kind=2) == I and _norm(kind=-1) == I
    assert _norm(xt=12) == U and b"x type 12" in lib().hy_last_error() and _norm(ot=8) == U
    assert _norm(m=-1) == I and _norm(n=0) == S and _norm(n=(1 << 22) + 1) == S and _norm(m=(1 << 30) + 1) == S
    assert _norm(x=None) == I and _norm(w=None) == I and _norm(out=None) == I
    assert _norm(x=TWO) == S and _norm(xt=BF16, x=ODD) == S and _norm(out=ODD) == S and _norm(out32=TWO, ld32=64) == S
    assert _norm(add=TWO, lda=64) == S and _norm(total=TWO, ldt=64) == S and _norm(w=TWO) == S and _norm(b=TWO) == S and _norm(mean=TWO) == S
    assert _norm(ldx=-1) == S and _norm(ldo=63) == S and _norm(total=P, ldt=63) == S and _norm(out32=P, ld32=0) == S
    assert _norm(eps=-1.0) == I and _norm(eps=float("nan")) == I
    assert _norm(m=0, x=None, out=None) == OK


def _bwd(kind=0, xt=F32, x=P, ldx=64, yt=BF16, dy=P, ldy=64, w=P, mean=P, rstd=P, resid=None, ldr=0, m=4, n=64, dx=P, ldd=64, dw=None, db=None,
         ws=None, wsb=0):
    return lib().hy_norm_bwd(kind, xt, x, ldx, yt, dy, ldy, w, mean, rstd, resid, ldr, m, n, dx, ldd, dw, db, 0, ws, wsb, None)


def test_norm_bwd_refusals():
    assert _bwd(kind=3) == I and _bwd(xt=2) == U and _bwd(yt=2) == U and b"dy type 2" in lib().hy_last_error()
    assert _bwd(m=-2) == I and _bwd(n=0) == S
    assert _bwd(x=None) == I and _bwd(dy=None) == I and _bwd(w=None) == I and _bwd(mean=None) == I and _bwd(rstd=None) == I and _bwd(dx=None) == I
    assert _bwd(dy=ODD) == S and _bwd(dx=TWO) == S and _bwd(rstd=TWO) == S and _bwd(resid=TWO, ldr=64) == S and _bwd(dw=TWO) == S and _bwd(ldd=10) == S
    assert _bwd(kind=1, mean=None, db=P) == I and b"no b" in lib().hy_last_error()
    need = lib().hy_norm_bwd_ws_bytes(1000, 64)
    assert need > 0 and lib().hy_norm_bwd_ws_bytes(1, 64) == 0 and lib().hy_norm_bwd_ws_bytes(0, 64) == 0 and lib().hy_norm_bwd_ws_bytes(8, 0) == 0
    assert _bwd(m=1000, dw=P) == I and b"workspace" in lib().hy_last_error()
    assert _bwd(m=1000, dw=P, ws=P, wsb=need - 1) == I and _bwd(m=1000, db=P, ws=ctypes.c_void_p(72), wsb=need) == S


def _route(logits=P, ls=64, E=64, bias=None, score=0, G=8, T=4, best=2, k=6, ids=P, wts=P, nt=3):
    return lib().hy_moe_route_groups(logits, ls, E, bias, score, G, T, best, k, 1, 1.0, ids, wts, nt, None)


def test_route_groups_refusals():
    assert _route(score=2) == I and _route(nt=-1) == I and _route(nt=1 << 24) == S
    assert _route(E=0) == S and _route(E=1025, G=1, T=1) == S and _route(k=0) == S and _route(k=65) == S
    assert _route(G=0) == S and _route(G=7) == S and _route(E=130, G=65) == S and _route(T=0) == S and _route(T=9) == S
    assert _route(best=0) == I and _route(best=3) == I
    assert _route(E=8, G=8, T=4, best=2, k=2) == S and b"2 best" in lib().hy_last_error()   # one expert a group
    assert _route(k=33) == S                                                                # more than the kept groups hold
    assert _route(logits=None) == I and _route(ids=None) == I and _route(wts=None) == I and _route(bias=TWO) == S and _route(ls=-1) == S
    assert _route(nt=0, logits=None, ids=None, wts=None) == OK


def test_route_groups_bwd_refusals():
    def call(logits=P, E=64, score=1, ids=P, k=6, dwts=P, dl=P, ty=BF16, ldd=64, nt=3):
        return lib().hy_moe_route_groups_bwd(logits, 64, E, score, ids, k, 1, 1.0, dwts, dl, ty, ldd, nt, None)
    assert call(score=5) == I and call(E=2000) == S and call(k=0) == S and call(nt=-1) == I and call(ty=9) == U
    assert call(logits=None) == I and call(ids=None) == I and call(dwts=None) == I and call(dl=None) == I
    assert call(dl=ODD) == S and call(ty=F32, dl=TWO) == S and call(ldd=63) == S and call(nt=0, logits=None) == OK


def _lora(ty=BF16, A=P, B=P, scale=None, nl=4, r=16, k=64, n=64, x=P, ldx=64, m=8, ids=P, resid=None, ldr=0, out=P, ot=BF16, ldo=64, ws=P, wsb=1 << 30):
    return lib().hy_lora(ty, A, B, scale, nl, r, k, n, x, ldx, m, ids, resid, ldr, out, ot, ldo, ws, wsb, None)


def test_lora_refusals():
    assert _lora(ty=F32) == U and _lora(ot=F16) == U and _lora(m=-1) == I and _lora(n=0) == S and _lora(k=0) == S
    assert _lora(nl=0) == I and _lora(r=0) == S and _lora(r=257) == S and b"rank 257" in lib().hy_last_error()
    assert _lora(A=None) == I and _lora(B=None) == I and _lora(x=None) == I and _lora(out=None) == I and _lora(ids=None) == I
    assert _lora(A=ODD) == S and _lora(out=TWO, ot=F32) == S and _lora(scale=TWO) == S and _lora(resid=ODD, ldr=64) == S and _lora(ldo=8) == S and _lora(ldx=-8) == S
    need = lib().hy_lora_ws_bytes(8, 16, 64)
    assert need == 8 * 16 * 4 and lib().hy_lora_ws_bytes(0, 16, 64) == 0 and lib().hy_lora_ws_bytes(8, 300, 64) == 0
    assert _lora(ws=None) == I and _lora(wsb=need - 1) == I and _lora(ws=ctypes.c_void_p(72)) == S
    assert _lora(m=1 << 28, n=1 << 14, ldo=1 << 14, wsb=1 << 45) == S and _lora(n=1 << 25, ldo=1 << 25) == S
    assert _lora(ldo=(1 << 22) + 1) == S and _lora(resid=P, ldr=(1 << 22) + 1) == S and b"2^22" in lib().hy_last_error()
    assert _lora(m=0, x=None, out=None, ids=None, ws=None) == OK


def test_long_contractions_and_batches_keep_their_parts_within_the_workspace():
    """the parts cover the contraction, none is empty, and there are at most 32"""
    for m in (1, 16, 17, 100, 4096, 1 << 20, 1 << 30):
        for k in (1, 255, 256, 257, 4096, 7168, 1 << 20, 1 << 30):
            splits = lib().hy_lora_ws_bytes(m, 1, k) // (4 * m)
            assert 1 <= splits <= 32 and lib().hy_lora_ws_bytes(m, 7, k) == splits * m * 7 * 4


def test_wrappers_refuse():
    f = lambda *s, dt=torch.float32: torch.zeros(*s, dtype=dt)  # noqa: E731
    x, w = f(4, 8), f(8)
    with pytest.raises(ValueError, match="unknown norm"):
        mm16.norm(x, w, f(4, 8), kind="batch")
    with pytest.raises(ValueError, match="add must be"):
        mm16.norm(x, w, f(4, 8), add=f(4, 8, dt=torch.bfloat16))
    with pytest.raises(ValueError, match="out must be"):
        mm16.norm(x, w, f(4, 9))
    with pytest.raises(ValueError, match="w must hold"):
        mm16.norm(x, f(7), f(4, 8))
    with pytest.raises(ValueError, match="float32, bfloat16 or float16"):
        mm16.norm(f(4, 8, dt=torch.float64), w, f(4, 8))
    with pytest.raises(ValueError, match="on a GPU"):
        mm16.norm(x, w, f(4, 8))
    with pytest.raises(ValueError, match="are needed"):
        mm16.norm_bwd(x, x, w, f(4), f(4, 8))
    with pytest.raises(ValueError, match="rstd must hold"):
        mm16.norm_bwd(x, x, w, f(3), f(4, 8), kind="rms")
    with pytest.raises(ValueError, match="unknown score"):
        mm16.route_groups(x, f(4, 2, dt=torch.int32), f(4, 2), score="relu")
    with pytest.raises(ValueError, match="ids must be"):
        mm16.route_groups(x, f(4, 2), f(4, 2))
    with pytest.raises(ValueError, match="wts must be"):
        mm16.route_groups(x, f(4, 2, dt=torch.int32), f(4, 3))
    with pytest.raises(ValueError, match="bias must hold"):
        mm16.route_groups(x, f(4, 2, dt=torch.int32), f(4, 2), bias=f(7))
    with pytest.raises(ValueError, match="dlogits must be"):
        mm16.route_groups_bwd(x, f(4, 2, dt=torch.int32), f(4, 2), f(4, 7))
    h = lambda *s: f(*s, dt=torch.bfloat16)  # noqa: E731
    with pytest.raises(ValueError, match="A must be"):
        mm16.Lora16(h(2, 4, 8), h(2, 16, 5))
    with pytest.raises(ValueError, match="of one type"):
        mm16.Lora16(h(2, 4, 8), f(2, 16, 4))
    with pytest.raises(ValueError, match="scale must hold"):
        mm16.Lora16(h(2, 4, 8), h(2, 16, 4), f(1))
    L = mm16.Lora16(h(2, 4, 8), h(2, 16, 4))
    with pytest.raises(ValueError, match="x must be"):
        mm16.lora(L, h(3, 9), f(3, dt=torch.int32), h(3, 16))
    with pytest.raises(ValueError, match="ids must hold"):
        mm16.lora(L, h(3, 8), f(2, dt=torch.int32), h(3, 16))
    with pytest.raises(ValueError, match="resid must be"):
        mm16.lora(L, h(3, 8), f(3, dt=torch.int32), h(3, 16), resid=f(3, 16))


def test_in_place_with_another_layout_is_refused():
    """another row would be overwritten before it is read"""
    q = ctypes.c_void_p(4096)
    assert _norm(out=P, ot=BF16) == S and b"out takes the place of x" in lib().hy_last_error()
    assert _norm(out=P, ot=F32, ldo=72) == S and _norm(xt=BF16, out=None, out32=P, ld32=64) == S and _norm(out=q, total=P, ldt=65) == S
    assert _norm(out=q, add=q, lda=64, total=q, ldt=66) == S and b"place of add" in lib().hy_last_error()
    assert _norm(out=P, ot=BF16, m=1) == S
    assert _norm(x=P, ldx=0, out=P, ot=F32) == S
    assert _bwd(dx=P, x=P, ldd=64, ldx=128, dy=q) == S and b"place of x" in lib().hy_last_error()
    assert _bwd(x=q, dy=P, yt=BF16, dx=P) == S and b"place of dy" in lib().hy_last_error()
    assert _bwd(x=q, dy=P, yt=F32, ldy=80, dx=P) == S and _bwd(x=q, dy=q, resid=P, ldr=0, dx=P) == S and b"place of resid" in lib().hy_last_error()
    assert _lora(out=q, resid=q, ldr=128) == S and b"place of resid" in lib().hy_last_error()
