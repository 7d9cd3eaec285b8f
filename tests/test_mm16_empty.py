"""Calls of the 16-bit expert products without pairs: the arrays may have no address, as empty tensors have."""
import ctypes

import hyper_amd
from hyper_amd import lib
from tests.test_mm16_args import BF16, F32, P, _dev

OK, I, S, U = hyper_amd.HY_OK, hyper_amd.HY_EINVAL, hyper_amd.HY_EBAD_SHAPE, hyper_amd.HY_EUNSUPPORTED_TYPE


def test_no_pairs_need_no_arrays():
    L, m = lib(), ctypes.byref(_dev())
    for max_active in (0, 4):
        assert L.hy_moe16_gate_up(m, None, 64, 2, None, 0, None, None, None, max_active, None, None, None, None) == OK
        assert L.hy_moe16_gate_up(m, None, 64, 2, None, 0, None, P, P, max_active, None, None, None, None) == OK
        assert L.hy_moe16_down(m, None, None, 0, None, None, None, max_active, None, None, F32, None) == OK
        assert L.hy_moe16_down_dx(m, None, 64, 2, 0, None, P, P, max_active, None, BF16, None) == OK
        assert L.hy_moe16_gate_up_dx(m, None, None, 0, None, P, P, max_active, None, BF16, None) == OK
    assert L.hy_swiglu_bwd(BF16, None, None, None, None, 0, 96, 0.0, None, None, None, None, None, None, None) == OK


def test_their_other_arguments_are_checked():
    L = lib()
    assert L.hy_moe16_gate_up(None, None, 64, 2, None, 0, None, None, None, 0, None, None, None, None) == I
    assert L.hy_moe16_gate_up(ctypes.byref(_dev(t=12)), None, 64, 2, None, 0, None, None, None, 0, None, None, None, None) == U
    m = ctypes.byref(_dev())
    assert L.hy_moe16_down_dx(m, None, 64, 0, 0, None, None, None, 0, None, BF16, None) == S
    assert L.hy_moe16_dw(m, BF16, None, 96, 1, 96, None, 64, 2, 64, 0, None, None, None, 0, None, F32, 0, None) == I    # dW is written
    assert L.hy_moe16_dw(m, BF16, None, 96, 1, 0, None, 64, 2, 64, 0, None, None, None, 0, P, F32, 0, None) == S
