"""linear_dw's workspace: asked for where the sum over the rows is cut into parts, and only there."""
import pytest
import torch

from hyper_amd import mm16
from tests.helpers import gen

LONG = [(8192, 264, 264), (65536, 64, 2048), (4096, 128, 128)]


def test_sizes_that_are_not_cut_need_none():
    for m, n, k in LONG:
        assert mm16.linear_dw_ws_bytes(m, n, k) >= 2 * 4 * (n * k + n)     # at least two parts
        for odd in ((m, n - 1, k), (m, n, k - 1), (m, n + 4, k), (m, n + 1, k + 3)):
            assert mm16.linear_dw_ws_bytes(*odd) == 0, odd
    assert mm16.linear_dw_ws_bytes(0, 64, 64) == 0 and mm16.linear_dw_ws_bytes(1, 64, 64) == 0


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("m,n,k", [(8192, 263, 264), (8192, 264, 263), (16384, 63, 129)])
def test_long_sums_of_odd_rows_without_one(cuda, dtype, m, n, k):
    g = gen(m + n)
    dz, x = torch.randint(-3, 4, (m, n), generator=g), torch.randint(-3, 4, (m, k), generator=g)
    dW, db = torch.empty(n, k, device=cuda), torch.empty(n, device=cuda)
    mm16.linear_dw(dz.to(dtype).to(cuda), x.to(dtype).to(cuda), dW, db=db)
    assert torch.equal(dW.cpu().double(), dz.double().t() @ x.double()) and torch.equal(db.cpu().double(), dz.double().sum(0))
