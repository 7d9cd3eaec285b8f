"""hy_moe16_reduce's argument checks, which come before any device work."""
import ctypes

import pytest
import torch

import hyper_amd
from hyper_amd import lib, mm16
from tests.test_mm16_args import P, _dev

I, S = hyper_amd.HY_EINVAL, hyper_amd.HY_EBAD_SHAPE


def test_refusals():
    def call(m=None, shexp=None, sg=None, y=P, k=2, out=P, nt=4, ids=P):
        return lib().hy_moe16_reduce(ctypes.byref(m or _dev()), shexp, sg, y, k, out, nt, ids, None)
    assert lib().hy_moe16_reduce(None, None, None, P, 2, P, 4, P, None) == I
    m = _dev()
    m.slot = None
    assert call(m) == I and call(y=None) == I and call(out=None) == I and call(ids=None) == I and call(nt=-1) == I
    assert call(k=0) == S and call(k=65) == S and call(nt=1 << 30) == S and b"2^30" in lib().hy_last_error()
    off = ctypes.c_void_p(66)
    assert call(y=off) == S and call(out=off) == S and call(ids=off) == S and call(shexp=off) == S and call(shexp=P, sg=off) == S
    assert call(nt=0, y=None, out=None, ids=None) == hyper_amd.HY_OK


def test_python_checks():
    b = torch.zeros(2, 8, 16, dtype=torch.bfloat16)
    m = mm16.Moe16Dev(b, b, None, torch.arange(2, dtype=torch.int32))
    ids = torch.zeros(6, dtype=torch.int32)
    for y, out, i in ((torch.zeros(5, 16), torch.zeros(3, 16), ids), (torch.zeros(6, 16), torch.zeros(3, 15), ids), (torch.zeros(6, 16).half(), torch.zeros(3, 16), ids),
                      (torch.zeros(6, 16), torch.zeros(3, 16), ids[:5]), (torch.zeros(6, 16), torch.zeros(3, 16), ids.long())):
        with pytest.raises(ValueError):
            mm16.moe16_reduce(m, None, None, y, 2, out, 3, i)
    with pytest.raises(ValueError, match="on a GPU"):
        mm16.moe16_reduce(m, None, None, torch.zeros(6, 16), 2, torch.zeros(3, 16), 3, ids)
