"""Low-rank adapters of many requests against 64-bit products.

With small integers every product and sum is exact (low products below 2^16, which two 16-bit values hold whole; sums below 2^24),
so a float32 output equals the formula's bit for bit and a 16-bit output is its nearest value.  With other values the bound
counts: (k + 40) 2^-23 sum |A x| for the low products (a unit in the last place a term, whether sums round or truncate, and the parts'
joins), twice half a step of the type squared for the two values that stand for one, (2 r + 4) 2^-23 sum |B low| for the second
product, 4 * 2^-24 for scale and residual, and half a step of the output's type."""
import pytest
import torch

from hyper_amd import mm16
from tests.helpers import gen
from tests.test_gpu_mm16 import empty, ints, put, same, within

pytestmark = pytest.mark.gpu
F32, BF, FP = torch.float32, torch.bfloat16, torch.float16
NAN = float("nan")


def lora64(A, B, scale, x, ids, resid):
    out = torch.zeros(x.shape[0], B.shape[1], dtype=torch.float64) if resid is None else resid.clone()
    for t, a in enumerate(ids.tolist()):
        if 0 <= a < A.shape[0]:
            out[t] += scale[a] * (B[a] @ (A[a] @ x[t]))
    return out


def workspace(L, m, dev):
    return torch.full((mm16.lora_ws_bytes(L, m),), 255, dtype=torch.uint8, device=dev)   # NaN as floats


def flat(t, dtype, dev, offset):
    """contiguous, `offset` elements off an aligned start"""
    buf = torch.full((t.numel() + offset,), NAN, dtype=dtype, device=dev)
    v = buf[offset:].view(t.shape)
    v.copy_(t.to(dtype))
    return v


def check_ints(m, k, n, r, n_a, dt, ot, ids, dev, seed, with_resid=True, with_scale=True, pad=0, offset=0, in_place=False):
    g = gen(seed)
    A, B, x = ints(g, n_a, r, k, lo=-1, hi=1), ints(g, n_a, n, r, lo=-2, hi=2), ints(g, m, k, lo=-2, hi=2)
    scale = 2.0 ** torch.randint(-1, 2, (n_a,), generator=g).double() if with_scale else torch.ones(n_a, dtype=torch.float64)
    resid = ints(g, m, n) if with_resid else None
    L = mm16.Lora16(flat(A, dt, dev, offset), flat(B, dt, dev, offset), scale.float().to(dev) if with_scale else None)
    out, around = empty(m, n, ot, dev, pad, offset)
    if in_place:
        out.copy_(resid.to(ot))
    mm16.lora(L, put(x, dt, dev, pad, offset), ids.to(dev), out, resid=out if in_place else put(resid, ot, dev, pad, offset) if with_resid else None,
              ws=workspace(L, m, dev))
    same(out, lora64(A, B, scale, x, ids, resid), f"m {m} k {k} n {n} r {r} adapters {n_a} {dt} {ot}")
    around()


def some_ids(g, m, n_a, how):
    if how == "each":
        return torch.randint(-1, n_a + 1, (m,), generator=g).to(torch.int32)   # -1 and n_a: none
    cuts = torch.sort(torch.randint(0, m + 1, (3,), generator=g)).values
    run = torch.bucketize(torch.arange(m), cuts, right=True)
    return torch.randint(-1, n_a, (4,), generator=g)[run].to(torch.int32)


@pytest.mark.parametrize("dt", [BF, FP])
@pytest.mark.parametrize("r", [1, 4, 8, 15, 16, 17, 20, 32, 33, 40, 64, 65, 96, 128, 200, 256])
def test_lora_ranks(r, dt):
    dev = torch.device("cuda:0")
    for i, (m, k, n, how) in enumerate(((1, 256, 256, "each"), (7, 100, 72, "each"), (33, 264, 300, "runs"), (70, 512, 64, "each"), (300, 200, 130, "runs"))):
        g = gen(r * 17 + i)
        check_ints(m, k, n, r, 5, dt, F32 if i % 2 else dt, some_ids(g, m, 5, how), dev, r + i, with_resid=i != 2, with_scale=i != 3,
                   pad=(0, 3, 8, 0, 1)[i], offset=(0, 1, 8, 0, 0)[i])


@pytest.mark.parametrize("k", [1, 2, 8, 63, 64, 72, 255, 256, 257, 520, 1024, 4096, 7168])
def test_lora_contractions(k):
    """lengths inside a product's step, a wave's turn and a part, and the parts' ends"""
    dev = torch.device("cuda:0")
    for i, m in enumerate((1, 16, 40)):
        check_ints(m, k, 96, 16, 3, (BF, FP)[i % 2], F32, some_ids(gen(k + i), m, 3, "each"), dev, k + i)


@pytest.mark.parametrize("n", [1, 3, 8, 15, 16, 63, 64, 65, 255, 256, 257, 1000, 7168])
def test_lora_outputs(n):
    dev = torch.device("cuda:0")
    for i, m in enumerate((1, 20, 260)):
        check_ints(m, 64, n, (8, 20, 48)[i], 3, (FP, BF)[i % 2], (F32, BF, FP)[i], some_ids(gen(n + i), m, 3, ("each", "runs", "runs")[i]), dev, n + i)


@pytest.mark.parametrize("m", [1, 2, 15, 16, 17, 63, 64, 65, 255, 256, 257, 1000, 2100])
def test_lora_rows(m):
    """single tokens with an adapter each, and prompts whose ends fall inside tiles"""
    dev = torch.device("cuda:0")
    for how in ("each", "runs"):
        check_ints(m, 320, 200, 16, 40 if how == "each" else 4, BF, F32, some_ids(gen(m), m, 40 if how == "each" else 4, how), dev, m)
        check_ints(m, 96, 264, 64, 9, FP, FP, some_ids(gen(m + 1), m, 9, how), dev, m, in_place=True)


@pytest.mark.parametrize("r", [8, 20, 64, 72])
def test_lora_many_rows_of_mixed_requests(r):
    """a large batch of single tokens: every tile has many adapters; odd and whole columns, both outputs, with and without a residual"""
    dev = torch.device("cuda:0")
    for i, (n, ot) in enumerate(((264, BF), (257, F32), (200, F32), (97, BF))):
        ids = some_ids(gen(r + i), 300 + 57 * i, 23, "each")
        check_ints(ids.numel(), 130, n, r, 23, BF, ot, ids, dev, r + i, with_resid=i != 2, pad=(0, 1)[i % 2], in_place=i == 1)


def test_lora_ends_of_the_matrices():
    """the last rows of the last adapter with nothing behind them: ranks and columns of every remainder"""
    dev = torch.device("cuda:0")
    for r in (1, 3, 7, 12, 31, 33, 63):
        for n in (1, 5, 64, 66):
            ids = torch.full((20,), 1, dtype=torch.int32)
            check_ints(20, 40, n, r, 2, FP, F32, ids, dev, r + n)
            check_ints(260, 40, n, r, 2, BF, BF, torch.full((260,), 1, dtype=torch.int32), dev, r + n)


def test_lora_no_adapters_and_no_rows():
    dev = torch.device("cuda:0")
    ids = torch.full((50,), -1, dtype=torch.int32)
    for in_place in (False, True):
        check_ints(50, 64, 72, 8, 2, BF, BF, ids, dev, 1, in_place=in_place)
    check_ints(50, 64, 72, 8, 2, BF, F32, ids, dev, 2, with_resid=False)
    check_ints(50, 64, 72, 8, 2, BF, F32, torch.tensor([-2 ** 31, 2 ** 31 - 1] * 25, dtype=torch.int32), dev, 3)
    L = mm16.Lora16(torch.zeros(1, 8, 64, dtype=BF, device=dev), torch.zeros(1, 72, 8, dtype=BF, device=dev))
    mm16.lora(L, torch.empty(0, 64, dtype=BF, device=dev), torch.empty(0, dtype=torch.int32, device=dev), torch.empty(0, 72, dtype=BF, device=dev))


@pytest.mark.parametrize("dt", [BF, FP])
def test_lora_values(dt):
    """random values of uneven rows, those near the ends of fp16's range among them"""
    dev = torch.device("cuda:0")
    for m, k, n, r, scale_x in ((5, 4096, 512, 16, 1.0), (300, 1000, 264, 64, 30.0), (40, 2048, 100, 200, 1e-3), (16, 512, 128, 8, 2000.0), (9, 256, 64, 16, 2.0 ** -14)):
        g = gen(m + k)
        rnd = lambda *s, mul: (torch.randn(*s, generator=g) * mul).to(dt).double()  # noqa: E731
        A, B = rnd(3, r, k, mul=k ** -0.5), rnd(3, n, r, mul=r ** -0.5)
        if scale_x == 2000.0:
            A *= 64   # low products beyond 65504
        x = rnd(m, k, mul=scale_x)
        scale = (0.5 + torch.rand(3, generator=g)).double() / (64 * scale_x if scale_x == 2000.0 else 1)
        scale = scale.float().double()
        resid = torch.randn(m, n, generator=g).double()
        ids = torch.randint(-1, 3, (m,), generator=g).to(torch.int32)
        L = mm16.Lora16(A.to(dt).to(dev), B.to(dt).to(dev), scale.float().to(dev))
        out = torch.empty(m, n, device=dev)
        mm16.lora(L, x.to(dt).to(dev), ids.to(dev), out, resid=resid.float().to(dev), ws=workspace(L, m, dev))
        resid = resid.float().double()
        want = lora64(A, B, scale, x, ids, resid)
        err = torch.zeros_like(want)
        half = (torch.finfo(dt).eps / 2) ** 2
        for t, a in enumerate(ids.tolist()):
            if a < 0:
                continue
            mag = A[a].abs() @ x[t].abs()
            low_err = (k + 40) * 2.0 ** -23 * mag + 2 * half * (A[a] @ x[t]).abs() + 2.0 ** -24 * half * (A[a] @ x[t]).abs().max()
            err[t] = scale[a] * (B[a].abs() @ low_err + (2 * r + 4) * 2.0 ** -23 * (B[a].abs() @ mag)) + 4 * 2.0 ** -24 * (want[t].abs() + resid[t].abs())
        within(out, want, err, f"{m} {k} {n} {r} {scale_x}")


def test_lora_other_requests_matrices_do_not_reach_a_row():
    """NaN and infinities in one adapter, and in one request's rows, stay with that request's rows; adapters nobody uses are not read"""
    dev = torch.device("cuda:0")
    g = gen(11)
    for m, r, k, n in ((16, 16, 256, 128), (70, 40, 300, 96), (300, 64, 128, 72)):
        A, B, x = ints(g, 4, r, k), ints(g, 4, n, r), ints(g, m, k)
        ids = torch.randint(0, 3, (m,), generator=g).to(torch.int32)
        A[2], B[2, :, 0], A[3], B[3] = NAN, float("inf"), NAN, NAN
        x[3] = float("inf")
        x[4, 7] = NAN
        ids[3] = ids[4] = 0
        L = mm16.Lora16(A.to(BF).to(dev), B.to(BF).to(dev))
        out = torch.empty(m, n, device=dev)
        mm16.lora(L, x.to(BF).to(dev), ids.to(dev), out, ws=workspace(L, m, dev))
        good = ((ids != 2) & (torch.arange(m) != 3) & (torch.arange(m) != 4)).nonzero()[:, 0]
        want = lora64(A, B, torch.ones(4, dtype=torch.float64), x, ids, None)
        same(out[good.to(dev)], want[good])
        assert out[4].isnan().all() and out[(ids == 2).to(dev)].isnan().all()


def test_lora_beside_a_projection_captured_replayed_and_on_another_stream():
    """linear with the adapters' sum into its output, in place, in a graph and on a stream of its own: the eager bits"""
    dev = torch.device("cuda:0")
    m, k, n, r = 24, 512, 384, 16
    g = gen(2)
    W = (torch.randn(n, k, generator=g) * k ** -0.5).to(BF).to(dev)
    L = mm16.Lora16((torch.randn(6, r, k, generator=g) * k ** -0.5).to(BF).to(dev), torch.randn(6, n, r, generator=g).to(BF).to(dev))
    x, ids = torch.empty(m, k, dtype=BF, device=dev), torch.empty(m, dtype=torch.int32, device=dev)
    ws = workspace(L, m, dev)

    def step(out, stream=None):
        mm16.linear(W, x, out, stream=stream)
        mm16.lora(L, x, ids, out, resid=out, ws=ws, stream=stream)

    def fill(seed):
        x.copy_(torch.randn(m, k, generator=gen(seed)))
        ids.copy_(torch.randint(-1, 6, (m,), generator=gen(seed + 1)))
    a, b, c = (torch.empty(m, n, device=dev) for _ in range(3))
    fill(1)
    step(b)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step(b)
    for seed in range(4):
        fill(10 + 5 * seed)
        step(a)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        s = torch.cuda.Stream()
        step(c, s)
        s.synchronize()
        assert torch.equal(a, b) and torch.equal(a, c)


@pytest.mark.parametrize("dt", [BF, FP])
@pytest.mark.parametrize("r", [8, 20, 33, 64, 72, 96, 160, 192, 200, 224])
def test_lora_columns_and_adapters_do_not_meet(r, dt):
    """what is not finite in one column of B stays in that column, and in its adapter, where a row of B is read past its ranks:
    whole multiples of 32 ranks that are fewer than the kernel takes among them"""
    dev = torch.device("cuda:0")
    for i, (m, k, n, resid) in enumerate(((6, 64, 72, False), (20, 64, 65, True), (40, 40, 128, True), (300, 64, 66, False))):
        g = gen(r + 50 * i)
        A, B, x = ints(g, 3, r, k, lo=-1, hi=1), ints(g, 3, n, r, lo=-2, hi=2), ints(g, m, k, lo=-2, hi=2)
        res = ints(g, m, n) if resid else None
        ids = (torch.arange(m) % 2).to(torch.int32)   # adapter 2 has no rows
        want = lora64(A, B, torch.ones(3, dtype=torch.float64), x, ids, res)
        bad = torch.zeros(m, n, dtype=torch.bool)
        B = B.clone()
        B[0, 5], B[1, 0], B[2, 0] = NAN, NAN, float("inf")
        bad[0::2, 5], bad[1::2, 0] = True, True
        L = mm16.Lora16(B=B.to(dt).to(dev), A=A.to(dt).to(dev))
        out = torch.full((m, n), 7.0, device=dev)
        mm16.lora(L, x.to(dt).to(dev), ids.to(dev), out, resid=res.float().to(dev) if resid else None, ws=workspace(L, m, dev))
        out = out.cpu()
        assert out[bad].isnan().all()
        same(out.where(~bad, torch.zeros(())), want.where(~bad, torch.zeros((), dtype=torch.float64)), f"rank {r} {dt} case {i}")
