"""Norms of rows that lie far from 0 beside their spread, and of constant rows, against 64-bit formulas.

Bounds that do not grow with the mean's size beyond what 64-bit sums and a mean of two floats leave.  With u = 2^-24, d the longest
chain of additions (at most 88, or 88 + n / 1024 above 16384 values) and D = s - mean:
  the mean used    half a step of its second float, u^2 |mean|, and (d + 2) 2^-53 mean |s| of its sum: e = 2 u^2 |mean| + (d + 2) 2^-53 mean |s|
  D                e and three roundings: the difference from the first float, at most u (|D| + u |mean|), and that from the second:
                   2 u |D| + u^2 |mean| + e
  rstd             half of the relative error of the variance, (d + 4) u of its sum and twice that of D in each term
                   (2 u |D| + f with f = u^2 |mean| + e: 4 u + 2 f / root(var) + f^2 / var), and 3 u of root, quotient and eps
  y                |D rstd w| (rstd's relative error + 4 u) + (2 u |D| + f) rstd |w| + 2 u |y|, and half a step of y's type
  mean             e and half a step"""
import pytest
import torch

from hyper_amd import mm16
from tests.helpers import gen
from tests.test_gpu_mm16 import empty, put, same, within
from tests.test_gpu_norm import EPS, eps32, norm64, u

pytestmark = pytest.mark.gpu
F32, BF, FP = torch.float32, torch.bfloat16, torch.float16


def check(n, s, yt, dev, add=None, pad=0, offset=0, what=""):
    """rows s (+ add, both as they are in float32 or a 16-bit type) through a layer norm"""
    g = gen(n)
    m, xt = s.shape[0], s.dtype
    w, b = (1 + 0.2 * torch.randn(n, generator=g)).float(), (0.1 * torch.randn(n, generator=g)).float()
    out, around = empty(m, n, yt, dev, pad, offset)
    total = empty(m, n, xt, dev, pad, offset)[0] if add is not None else None
    mean, rstd = torch.full((m,), 7.0, device=dev), torch.full((m,), 7.0, device=dev)
    mm16.norm(put(s.double(), xt, dev, pad, offset), w.to(dev), out, b=b.to(dev), eps=EPS, add=None if add is None else put(add.double(), xt, dev, pad, offset),
              total=total, mean=mean, rstd=rstd)
    around()
    if add is not None:
        s = (s.float() + add.float()).to(xt)
        same(total, s.double(), what + " total")
    s, w, b = s.double(), w.double(), b.double()
    y, mu, r = norm64(s, w, b, True)
    D, d = (s - mu).abs(), 88 + (n // 1024 if n > 16384 else 0)
    e = 2 * u * u * mu.abs() + (d + 2) * 2.0 ** -53 * s.abs().mean(1, keepdim=True)
    f = u * u * mu.abs() + e
    within(mean[:, None], mu, e, what + " mean")
    r_rel = 0.5 * ((d + 8) * u + 2 * f * r + (f * r) ** 2) + 3 * u
    within(rstd[:, None], r, r * r_rel, what + " rstd")
    within(out, y, D * r * w.abs() * (r_rel + 4 * u) + (2 * u * D + f) * r * w.abs() + 2 * u * y.abs(), what)


@pytest.mark.parametrize("n", [7, 64, 640, 1001, 2047, 4096, 5000, 7168, 9001, 16384, 16390, 40001])
def test_layer_norm_of_rows_far_from_zero(n):
    dev = torch.device("cuda:0")
    g = gen(n)
    for i, (mean, sd) in enumerate(((100.0, 0.01), (1e5, 0.05), (-1000.0, 0.03), (3e-3, 1.0), (-7e6, 2.0))):
        s = (mean + sd * torch.randn(3, n, generator=g, dtype=torch.float64)).float()
        check(n, s, (F32, F32, BF, F32, F32)[i], dev, pad=i, offset=i % 3, what=f"{n} {mean} {sd}")
        check(n, s, F32, dev, add=(sd * torch.randn(3, n, generator=g)).float(), what=f"{n} {mean} {sd} add")
    # 16-bit rows of a few steps around their mean, y as the statistics leave it
    for xt, mean in ((FP, 1500.0), (BF, 100.0)):
        step = mean * torch.finfo(xt).eps
        s = (mean + step * torch.randint(-3, 4, (3, n), generator=g)).to(xt)
        check(n, s, F32, dev, what=f"{n} {xt}")


@pytest.mark.parametrize("n", [3, 5, 640, 1001, 2047, 5000, 9001, 16383, 20000, 65537])
def test_layer_norm_of_constant_rows(n):
    """the sum of n <= 2^22 equal floats has at most 24 + 22 digits: exact in 64 bits, so the mean is the value and nothing is left"""
    dev = torch.device("cuda:0")
    w = torch.rand(n, generator=gen(n)).to(dev)
    for c in (0.1, -1e4 / 3, 7e-30, 1e30, 3e38):
        out, mean, rstd = torch.empty(2, n, device=dev), torch.empty(2, device=dev), torch.empty(2, device=dev)
        x = torch.full((2, n), c, device=dev)
        mm16.norm(x, w, out, b=2 * w, eps=EPS, mean=mean, rstd=rstd)
        assert torch.equal(out, (2 * w).expand(2, n)) and torch.equal(mean, x[:, 0]), (n, c)
        assert (rstd - eps32 ** -0.5).abs().max() <= 400 * u
