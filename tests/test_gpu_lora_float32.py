"""Adapters into float32 outputs: nothing of a low product is lost.

Integers whose low products need up to 24 binary places (x and A as large as their type holds exactly, sums below 2^24), B of -1, 0
and 1 with as few entries a row as keep its sums below 2^24: every sum is exact in float32, so the output equals the formula's bit
for bit unless a low product was rounded on its way to B."""
import pytest
import torch

from hyper_amd import mm16
from tests.helpers import gen
from tests.test_gpu_lora import flat, lora64, some_ids, workspace
from tests.test_gpu_mm16 import empty, ints, put, same

pytestmark = pytest.mark.gpu
F32, BF, FP = torch.float32, torch.bfloat16, torch.float16


def check(m, k, n, r, dt, most, dev, seed, resid=False, in_place=False, pad=0, offset=0, how="each"):
    """A and x of up to `most`; k most^2 < 2^24"""
    g = gen(seed)
    few = (2 ** 24 - 1 - (1000 if resid else 0)) // (k * most * most)   # entries of a row of B
    assert few >= 1
    A, x = ints(g, 3, r, k, lo=-most, hi=most), ints(g, m, k, lo=-most, hi=most)
    x[::2] = x[::2].abs()   # rows of large low products
    A[0] = A[0].abs()
    B = torch.zeros(3, n, r, dtype=torch.float64)
    for _ in range(min(few, r)):
        B.scatter_(2, torch.randint(0, r, (3, n, 1), generator=g), 2.0 * torch.randint(0, 2, (3, n, 1), generator=g).double() - 1)
    res = ints(g, m, n, lo=-1000, hi=1000) if resid else None
    ids = some_ids(g, m, 3, how)
    L = mm16.Lora16(flat(A, dt, dev, offset), flat(B, dt, dev, offset))
    out, around = empty(m, n, F32, dev, pad, offset)
    if in_place:
        out.copy_(res.float())
    mm16.lora(L, put(x, dt, dev, pad, offset), ids.to(dev), out, resid=out if in_place else put(res, F32, dev, pad, offset) if resid else None,
              ws=workspace(L, m, dev))
    same(out, lora64(A, B, torch.ones(3, dtype=torch.float64), x, ids, res), f"m {m} k {k} n {n} r {r} {dt}")
    around()


@pytest.mark.parametrize("dt", [BF, FP])
@pytest.mark.parametrize("r", [1, 8, 20, 32, 64, 72, 128, 200, 256])
def test_lora_float32_keeps_the_low_products(r, dt):
    dev = torch.device("cuda:0")
    big = 255 if dt is BF else 1000   # low products of 24 places
    k = 256 if dt is BF else 16
    for i, (m, n, how) in enumerate(((1, 64, "runs"), (20, 65, "each"), (40, 264, "runs"), (300, 264, "runs"), (300, 72, "each"), (270, 97, "each"))):
        check(m, k, n, r, dt, big, dev, r + i, how=how, pad=(0, 3)[i % 2], offset=(0, 1)[i % 2])
        check(m, 64, n, r, dt, 100, dev, r + 7 * i, resid=True, in_place=i % 2 == 0, how=how)
