"""The 16-bit matrix products' argument checks, which come before any device work: codes and messages of the C entries, and
the Python wrappers' ValueErrors."""
import ctypes

import pytest
import torch

import hyper_amd
from hyper_amd import hy_moe_dev, lib, mm16

I, S, U = hyper_amd.HY_EINVAL, hyper_amd.HY_EBAD_SHAPE, hyper_amd.HY_EUNSUPPORTED_TYPE
P = ctypes.c_void_p(64)
ODD = ctypes.c_void_p(65)
BF16, F16, F32 = 30, 1, 0


def _linear(type_=BF16, W=P, ldw=64, n=64, k=64, x=P, ldx=64, m=8, bias=None, act=0, resid=None, ldr=0, z=None, ldz=0, out=P, ot=BF16, ldo=64):
    return lib().hy_linear(type_, W, ldw, n, k, x, ldx, m, bias, act, resid, ldr, z, ldz, out, ot, ldo, None)


def test_linear_refusals():
    assert _linear(type_=12) == U and b"type 12" in lib().hy_last_error()
    assert _linear(type_=F32) == U
    assert _linear(ot=F16) == U                                # neither the operands' type nor float32
    assert _linear(m=-1) == I and _linear(n=0) == S and _linear(k=0) == S and _linear(n=(1 << 30) + 1) == S
    assert _linear(W=None) == I and _linear(x=None) == I and _linear(out=None) == I
    assert _linear(W=ODD) == S and _linear(x=ODD) == S and _linear(out=ODD) == S
    assert _linear(out=ctypes.c_void_p(66), ot=F32) == S       # a float32 row off its 4 bytes
    assert _linear(act=5) == I and _linear(act=-1) == I
    assert _linear(ldo=63) == S and _linear(ldx=-1) == S
    assert _linear(resid=ODD, ldr=64) == S and _linear(z=P, ldz=32) == S and _linear(bias=ctypes.c_void_p(66)) == S
    assert _linear(m=0) == hyper_amd.HY_OK                     # nothing to do


def test_linear_glu_refusals():
    def call(type_=F16, Wg=P, Wu=P, n=64, m=8, g=None, u=None, h=P, ldh=64):
        return lib().hy_linear_glu(type_, Wg, Wu, 64, n, 64, P, 64, m, 0.0, g, u, h, ldh, None)
    assert call(type_=8) == U and call(Wu=None) == I and call(h=None) == I and call(ldh=10) == S
    assert call(g=P) == I and b"together" in lib().hy_last_error()
    assert call(g=P, u=ODD) == S and call(m=0) == hyper_amd.HY_OK


def test_linear_gradient_refusals():
    L = lib()
    assert L.hy_act_bwd(BF16, 9, P, 64, P, 64, 8, 64, P, 64, None) == I
    assert L.hy_act_bwd(BF16, 1, P, 64, P, 64, 8, 64, P, 8, None) == S
    assert L.hy_act_bwd(BF16, 1, P, 64, None, 64, 8, 64, P, 64, None) == I
    assert L.hy_linear_dx(BF16, P, 64, 64, 64, P, 64, 8, None, 0, None, BF16, 64, None) == I
    assert L.hy_linear_dx(BF16, P, 64, 64, 64, P, 64, 8, None, 0, P, F16, 64, None) == U
    assert L.hy_linear_dx(BF16, P, 64, 64, 64, P, 64, 0, None, 0, P, BF16, 64, None) == hyper_amd.HY_OK

    def dw(dz=P, m=64, n=64, k=64, dW=P, ot=F32, ldw=64, db=None, ws=None, wsb=0):
        return L.hy_linear_dw(BF16, dz, n, P, k, m, n, k, dW, ot, ldw, db, 0, ws, wsb, None)
    assert dw(dz=None) == I and dw(dW=None) == I and dw(ldw=63) == S and dw(ot=F16) == U and dw(m=-1) == I
    assert dw(db=ctypes.c_void_p(66)) == S
    big = dict(m=8192, n=128, k=128, ldw=128)   # a long sum over few tiles needs a workspace where the library splits it
    if L.hy_linear_dw_ws_bytes(8192, 128, 128):
        assert dw(**big) == I and b"workspace" in L.hy_last_error()
        assert dw(**big, ws=P, wsb=16) == I
        assert dw(**big, ws=ctypes.c_void_p(72), wsb=1 << 40) == S


def _dev(t=BF16, ff=96, n=64, E=4):
    m = hy_moe_dev()
    m.gate = m.up = m.down = m.slot = 64
    m.tg = m.td = t
    m.ff, m.n, m.n_expert, m.n_local = ff, n, E, E
    m.gate_bytes = m.down_bytes = 2 * ff * n
    return m


def test_expert_refusals():
    L = lib()

    def gate_up(m, k=2, ids=None, n_pairs=8, order=P, order_n=P, egrp=P, ma=4, g=None, u=None, h=P, x=P):
        return L.hy_moe16_gate_up(ctypes.byref(m), x, 64, k, ids, n_pairs, order, order_n, egrp, ma, g, u, h, None)
    assert gate_up(_dev(t=12)) == U                            # a quantized layer
    for field in ("gate", "up", "slot"):
        m = _dev()
        setattr(m, field, None)
        assert gate_up(m) == I, field
    m = _dev()
    m.gate_bytes += 2
    assert gate_up(m) == S and b"gate_bytes" in L.hy_last_error()
    m = _dev()
    m.up = 65
    assert gate_up(m) == S
    m = _dev()
    m.n_local = 0
    assert gate_up(m) == I
    assert gate_up(_dev(), k=0) == S and gate_up(_dev(), k=65) == S
    assert gate_up(_dev(), n_pairs=-1) == I and gate_up(_dev(), order_n=None) == I and gate_up(_dev(), egrp=None) == I
    assert gate_up(_dev(), ma=0) == S and gate_up(_dev(), ma=1025) == S
    assert gate_up(_dev(), order=None) == I                    # neither ids nor order
    assert gate_up(_dev(), order=None, ids=P, n_pairs=65536) == S
    assert gate_up(_dev(), g=P) == I and gate_up(_dev(), h=None) == I and gate_up(_dev(), x=ODD) == S
    assert gate_up(_dev(), n_pairs=0) == hyper_amd.HY_OK

    def down(m, ot=F32, wts=P, y=P):
        return L.hy_moe16_down(ctypes.byref(m), P, None, 8, P, P, P, 4, wts, y, ot, None)
    m = _dev()
    m.td = 14
    assert down(m) == U and down(_dev(), ot=F16) == U and down(_dev(), y=None) == I and down(_dev(), wts=ctypes.c_void_p(66)) == S

    assert L.hy_moe16_down_dx(ctypes.byref(_dev()), P, 64, 0, 8, P, P, P, 4, P, BF16, None) == S
    assert L.hy_moe16_down_dx(ctypes.byref(_dev()), P, 64, 2, 8, None, P, P, 4, P, BF16, None) == I
    assert L.hy_moe16_gate_up_dx(ctypes.byref(_dev()), P, None, 8, P, P, P, 4, P, BF16, None) == I

    def dw(rows=96, cols=64, ka=1, kb=2, dW=P, ot=F32, type_=BF16, n_pairs=8):
        return L.hy_moe16_dw(ctypes.byref(_dev()), type_, P, rows, ka, rows, P, cols, kb, cols, n_pairs, P, P, P, 4, dW, ot, 0, None)
    assert dw(rows=0) == S and dw(cols=0) == S and dw(ka=0) == S and dw(kb=65) == S and dw(dW=None) == I and dw(ot=F16) == U
    assert dw(type_=15) == U and dw(n_pairs=-1) == I

    def glu(g=P, order=None, order_n=None, wts=P, n_pairs=8, ff=96):
        return L.hy_swiglu_bwd(BF16, g, P, P, wts, n_pairs, ff, 0.0, order, order_n, P, P, None, None, None)
    assert glu(g=None) == I and glu(order=P) == I and glu(wts=ctypes.c_void_p(66)) == S and glu(ff=0) == S and glu(n_pairs=-1) == I
    assert L.hy_rows16(F32, P, 64, 64, 8, P, 64, None) == U and L.hy_rows16(BF16, P, 64, 64, 8, P, 32, None) == S


def test_upload_takes_plain_matrices_only_in_their_size():
    import numpy as np
    from hyper_amd import hy_expert_tensors
    L = lib()
    buf, sl, out, t = np.zeros(4096, np.uint8), np.zeros(1, np.int32), hy_moe_dev(), hy_expert_tensors()
    t.gate = t.up = t.down = buf.ctypes.data
    t.E, t.tg, t.td, t.gb, t.db = 1, BF16, F16, 2 * 24 * 16, 2 * 24 * 16 + 2
    call = lambda: L.hy_upload_experts(ctypes.byref(t), sl.ctypes.data_as(ctypes.c_void_p), 24, 16, 0.0, ctypes.byref(out))  # noqa: E731
    assert call() == S
    t.db, t.td = 2 * 24 * 16, 12                               # one side quantized: the tiled sizes apply
    assert call() in (S, U)


def test_python_checks():
    """ValueError before the library is called; CPU tensors are refused, not computed elsewhere."""
    b = lambda *s: torch.zeros(*s, dtype=torch.bfloat16)  # noqa: E731
    with pytest.raises(ValueError, match="on a GPU"):
        mm16.linear(b(8, 16), b(4, 16), b(4, 8))
    for bad in (dict(x=b(4, 15)), dict(out=b(4, 9)), dict(x=b(4, 16).half()), dict(W=torch.zeros(8, 16)), dict(act="swish"),
                dict(bias=b(8)), dict(bias=torch.zeros(7)), dict(resid=torch.zeros(4, 8)), dict(x=b(16, 4).t())):
        a = dict(dict(W=b(8, 16), x=b(4, 16), out=b(4, 8)), **bad)
        with pytest.raises(ValueError):
            mm16.linear(**a)
    with pytest.raises(ValueError):
        mm16.Moe16Dev(b(2, 8, 16), b(2, 8, 16), b(2, 16, 9), torch.zeros(2, dtype=torch.int32))
    with pytest.raises(ValueError):
        mm16.Moe16Dev(b(2, 8, 16), None, None, torch.zeros(2, dtype=torch.int32))
    with pytest.raises(ValueError):
        mm16.Moe16Dev(b(2, 8, 16), b(2, 8, 16), None, torch.zeros(2))
    m = mm16.Moe16Dev(b(2, 8, 16), b(2, 8, 16), None, torch.arange(2, dtype=torch.int32))
    with pytest.raises(ValueError, match="no down"):
        mm16.moe16_down(m, b(4, 8), 4, b(4, 16))
    with pytest.raises(ValueError):
        mm16.moe16_gate_up(m, b(2, 16), 2, 4, b(4, 9), ids=torch.zeros(4, dtype=torch.int32))
    with pytest.raises(ValueError):
        mm16.moe16_gate_up(m, b(1, 16), 2, 4, b(4, 8), ids=torch.zeros(4, dtype=torch.int32))     # four pairs are two rows
