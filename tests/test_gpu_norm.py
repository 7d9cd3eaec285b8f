"""Norms and their gradients against 64-bit formulas.

Bounds, with u = 2^-24 and d the longest chain of additions of a sum (a row's sums: at most 64 values a thread, 6 steps across a wave,
16 waves; rows above 16384 values: n / 1024 a thread; the sums over the rows: every row of a block's part, 8 rows of the block, 32
joined parts, 16 waves):  a sum of terms t is off by at most (d + 1) u sum |t|.  With s = x - mean:
  mean    (d + 2) u mean |x|
  rstd    half of the relative error of the variance, (d + 4) u + (mean's error)^2 / var, and 3 u of root, quotient and eps
  y       |s rstd w| (rstd's relative error + 4 u) + (mean's error) rstd |w| + 2 u |y|, and half a step of y's type
  dx      from given statistics: h and g = dy w are off by 3 u (|h| + |x| rstd) and u |g|; the two means by (d + 6) u of the means of
          absolute values;  all that times rstd, and 4 u of the terms' absolute values
  dw, db  (d + 4) u sum |dy h|  +  3 u sum |dy x| rstd,  (d + 1) u sum |dy|"""
import pytest
import torch

from hyper_amd import mm16
from tests.helpers import gen
from tests.test_gpu_mm16 import empty, put, same, within

pytestmark = pytest.mark.gpu
u = 2.0 ** -24
F32, BF, FP = torch.float32, torch.bfloat16, torch.float16
EPS = 1e-5
eps32 = float(torch.tensor(EPS, dtype=F32))


def rows(g, m, n, dtype):
    """uneven rows with an offset, as they are in `dtype` (64 bits)"""
    x = (torch.randn(m, n, generator=g) + 0.3) * torch.exp(0.5 * torch.randn(m, 1, generator=g))
    return x.to(dtype).double()


def depth(n):
    return 88 + (n // 1024 if n > 16384 else 0)


def norm64(s, w, b, layer):
    mean = s.mean(1, keepdim=True) if layer else torch.zeros(s.shape[0], 1, dtype=torch.float64)
    rstd = (((s - mean) ** 2).mean(1, keepdim=True) + eps32) ** -0.5
    y = (s - mean) * rstd * w
    return (y + b if b is not None else y), mean, rstd


def check_norm(kind, m, n, xt, yt, add, b, dev, seed, pad=0, offset=0, out32=False):
    g = gen(seed)
    layer = kind == "layer"
    x, w = rows(g, m, n, xt), (1 + 0.2 * torch.randn(n, generator=g)).float().double()
    bias = (0.1 * torch.randn(n, generator=g)).float().double() if b else None
    d = rows(g, m, n, xt) if add else None
    s = (x + d).to(F32).to(xt).double() if add else x
    out, around = empty(m, n, yt, dev, pad, offset)
    total, around_t = empty(m, n, xt, dev, pad, offset) if add else (None, lambda: None)
    o32, around32 = empty(m, n, F32, dev, pad, offset) if out32 else (None, lambda: None)
    mean, rstd = torch.full((m,), 7.0, device=dev), torch.full((m,), 7.0, device=dev)
    mm16.norm(put(x, xt, dev, pad, offset), w.float().to(dev), out, b=bias.float().to(dev) if b else None, eps=EPS, kind=kind,
              add=put(d, xt, dev, pad, offset) if add else None, total=total, out32=o32, mean=mean, rstd=rstd)
    what = f"{kind} {m}x{n} {xt} -> {yt} add {add} b {b}"
    if add:
        same(total, s, what + " total")
    y, mu, r = norm64(s, w, bias, layer)
    var = ((s - mu) ** 2).mean(1, keepdim=True) + eps32
    mu_err = (depth(n) + 2) * u * s.abs().mean(1, keepdim=True) if layer else torch.zeros_like(mu)
    r_rel = 0.5 * ((depth(n) + 4) * u + mu_err ** 2 / var) + 3 * u
    within(mean[:, None], mu, mu_err, what + " mean")
    within(rstd[:, None], r, r * r_rel, what + " rstd")
    err = ((s - mu) * r * w).abs() * (r_rel + 4 * u) + mu_err * r * w.abs() + 2 * u * y.abs()
    within(out, y, err, what)
    if out32:
        within(o32, y, err, what + " out32")
        around32()
    around()
    around_t()


WIDTHS = [1, 2, 7, 64, 65, 255, 512, 513, 1000, 1024, 1032, 2047, 2048, 2056, 4096, 4100, 7168, 8192, 8200, 16384, 16390, 40000]


@pytest.mark.parametrize("n", WIDTHS)
def test_norm_widths(n):
    """each width's kernel, 16-byte rows and odd ones, both kinds"""
    dev = torch.device("cuda:0")
    for seed, (kind, xt, yt, add, b, pad, offset) in enumerate([
            ("rms", F32, BF, True, False, 0, 0), ("layer", FP, FP, False, True, 0, 0), ("layer", F32, F32, True, True, 3, 1),
            ("rms", BF, F32, False, True, 1, 1), ("layer", BF, BF, True, False, 8, 8)]):
        check_norm(kind, 3, n, xt, yt, add, b, dev, seed + n, pad, offset, out32=seed % 2 == 0)


@pytest.mark.parametrize("n", [40, 640, 1000, 1600, 2048, 4096, 4104, 6000, 8192, 9000])
def test_norm_many_rows(n):
    """from 1024 rows on other numbers of threads share a row"""
    dev = torch.device("cuda:0")
    for seed, (kind, xt, yt, add, pad) in enumerate([("layer", F32, BF, False, 0), ("rms", FP, FP, True, 0), ("layer", BF, F32, True, 1)]):
        check_norm(kind, 1025, n, xt, yt, add, True, dev, seed + n, pad)


def test_norm_of_no_rows_and_constant_rows():
    dev = torch.device("cuda:0")
    w = torch.ones(64, device=dev)
    mm16.norm(torch.empty(0, 64, device=dev), w, torch.empty(0, 64, device=dev))
    for c in (0.0, 3.0, -1e4, 1e30):   # no variance: (s - mean) is 0 where the mean is exact, and 1 / sqrt(eps) scales it
        out, rstd = torch.empty(2, 64, device=dev), torch.empty(2, device=dev)
        mm16.norm(torch.full((2, 64), c, device=dev), w, out, b=2 * w, eps=EPS, rstd=rstd)
        assert (out == 2).all() and (rstd - eps32 ** -0.5).abs().max() <= 400 * u
    out = torch.empty(1, 64, device=dev)
    mm16.norm(torch.zeros(1, 64, device=dev), w, out, eps=0.0, kind="rms")   # 0 / 0
    assert out.isnan().all()


def test_norm_of_infinities_and_nan_stays_in_its_row():
    dev = torch.device("cuda:0")
    for n in (64, 1000, 5000, 20000):
        x = torch.randn(9, n, generator=gen(n))
        clean, dirty = torch.empty(9, n, device=dev, dtype=BF), torch.empty(9, n, device=dev, dtype=BF)
        w = torch.ones(n, device=dev)
        mm16.norm(x.to(dev), w, clean)
        x[2, n // 2], x[5, n - 1] = float("inf"), float("nan")
        mm16.norm(x.to(dev), w, dirty)
        assert dirty[2].isnan().any() and dirty[5].isnan().all()
        keep = [i for i in range(9) if i not in (2, 5)]
        assert torch.equal(clean[keep], dirty[keep])


def test_norm_in_place():
    """total may be x or add, out may be x: the same bits as apart"""
    dev = torch.device("cuda:0")
    for n in (7, 640, 4096, 20000):
        g = gen(n)
        x, d = torch.randn(5, n, generator=g).to(dev), torch.randn(5, n, generator=g).to(dev)
        w = torch.rand(n, generator=g).to(dev)
        total, out = torch.empty_like(x), torch.empty_like(x)
        mm16.norm(x, w, out, add=d, total=total)
        a, o = x.clone(), torch.empty_like(x)
        mm16.norm(a, w, o, add=d, total=a)
        assert torch.equal(a, total) and torch.equal(o, out)
        a = d.clone()
        mm16.norm(x, w, o, add=a, total=a)
        assert torch.equal(a, total) and torch.equal(o, out)
        a = total.clone()
        mm16.norm(a, w, a)
        assert torch.equal(a, out)


# ------------------------------------------------------------------ backward

def bwd64(x, dy, w, mu, r, resid, layer):
    h, g = (x - mu) * r, dy * w
    dx = g - h * (g * h).mean(1, keepdim=True)
    if layer:
        dx = dx - g.mean(1, keepdim=True)
    dx = dx * r
    return (dx if resid is None else dx + resid), (dy * h).sum(0), dy.sum(0)


def check_bwd(kind, m, n, xt, yt, resid, dev, seed, pad=0, offset=0, accumulate=False, want=(True, True)):
    g = gen(seed)
    layer = kind == "layer"
    x, dy = rows(g, m, n, xt), (0.1 * torch.randn(m, n, generator=g)).to(yt).double()
    w = (1 + 0.2 * torch.randn(n, generator=g)).float().double()
    e = rows(g, m, n, xt) if resid else None
    _, mu, r = norm64(x, w, None, layer)
    mu, r = mu.float().double(), r.float().double()
    dx, around = empty(m, n, xt, dev, pad, offset)
    dw, db = torch.full((n,), 0.25, device=dev) if want[0] else None, torch.full((n,), 0.25, device=dev) if layer and want[1] else None
    ws = torch.full((mm16.norm_bwd_ws_bytes(m, n),), 255, dtype=torch.uint8, device=dev)   # NaN as floats
    mm16.norm_bwd(put(x, xt, dev, pad, offset), put(dy, yt, dev, pad, offset), w.float().to(dev), r[:, 0].float().to(dev), dx,
                  mean=mu[:, 0].float().to(dev) if layer else None, kind=kind, resid=put(e, xt, dev, pad, offset) if resid else None,
                  dw=dw, db=db, accumulate=accumulate, ws=ws)
    what = f"{kind} {m}x{n} {xt} dy {yt} resid {resid}"
    ref, rw, rb = bwd64(x, dy, w, mu, r, e, layer)
    gw, h = (dy * w).abs(), (x - mu).abs() * r
    h_err = 3 * u * (h + x.abs() * r)
    d = 88 + n // 1024
    c2 = (gw * h).mean(1, keepdim=True)
    c2_err = (d + 6) * u * c2 + (gw * h_err).mean(1, keepdim=True)
    c1 = gw.mean(1, keepdim=True) if layer else torch.zeros_like(mu)
    err = r * (u * gw + h_err * c2 + h * c2_err + (d + 6) * u * c1 + 4 * u * (gw + h * c2 + c1))
    if resid:
        err = err + u * (e.abs() + ref.abs())
    within(dx, ref, err, what + " dx")
    around()
    d = m + 60   # (every row of a column in one chain, and the joins)
    start = 0.25 if accumulate else 0.0
    if dw is not None:
        bound = (d + 4) * u * (dy.abs() * h).sum(0) + (dy.abs() * h_err).sum(0) + u * (start + rw.abs())
        within(dw, rw + start, bound, what + " dw")
    if db is not None:
        within(db, rb + start, (d + 1) * u * dy.abs().sum(0) + u * (start + rb.abs()), what + " db")


@pytest.mark.parametrize("n", WIDTHS)
def test_norm_bwd_widths(n):
    dev = torch.device("cuda:0")
    for seed, (kind, m, xt, yt, resid, pad, offset) in enumerate([
            ("rms", 1, F32, BF, True, 0, 0), ("layer", 3, FP, FP, False, 0, 0), ("layer", 9, F32, F32, True, 3, 1), ("rms", 19, BF, BF, False, 1, 1),
            ("layer", 37, F32, FP, True, 0, 0)]):
        check_bwd(kind, m, n, xt, yt, resid, dev, seed + n, pad, offset, accumulate=seed % 2 == 1)


@pytest.mark.parametrize("m", [2, 8, 9, 511, 513, 4097, 5000])
def test_norm_bwd_rows(m):
    """blocks of one and of several turns, and joins of every length"""
    dev = torch.device("cuda:0")
    for seed, (kind, n, resid) in enumerate([("layer", 300, True), ("rms", 1100, False), ("layer", 4096, False), ("layer", 4500, True), ("rms", 9000, True)]):
        if m * n < 20e6:
            check_bwd(kind, m, n, F32 if seed % 2 else BF, BF, resid, dev, seed + m, accumulate=seed % 2 == 0, want=(seed != 3, seed != 0))


def test_norm_bwd_without_rows():
    dev = torch.device("cuda:0")
    none, w = torch.empty(0, 100, device=dev), torch.ones(100, device=dev)
    dw, db = torch.full((100,), 3.0, device=dev), torch.full((100,), 3.0, device=dev)
    e = torch.empty(0, device=dev)
    mm16.norm_bwd(none, none, w, e, none, mean=e, dw=dw, db=db, accumulate=True)
    assert (dw == 3).all() and (db == 3).all()
    mm16.norm_bwd(none, none, w, e, none, mean=e, dw=dw, db=db)
    assert (dw == 0).all() and (db == 0).all()


def test_norm_bwd_in_place():
    dev = torch.device("cuda:0")
    for n in (100, 4096, 7000, 9000):
        g = gen(n)
        x, dy, e = (torch.randn(40, n, generator=g).to(dev) for _ in range(3))
        w, r = torch.rand(n, generator=g).to(dev), torch.rand(40, generator=g).to(dev)
        ws = torch.empty(mm16.norm_bwd_ws_bytes(40, n), dtype=torch.uint8, device=dev)

        def call(x, dy, dx, e):
            dw = torch.empty(n, device=dev)
            mm16.norm_bwd(x, dy, w, r, dx, kind="rms", resid=e, dw=dw, ws=ws)
            return dw
        dx = torch.empty_like(x)
        dw = call(x, dy, dx, e)
        for name in ("x", "dy", "e"):
            t = {"x": x, "dy": dy, "e": e}
            t[name] = t[name].clone()
            assert torch.equal(call(t["x"], t["dy"], t[name], t["e"]), dw) and torch.equal(t[name], dx), (n, name)


@pytest.mark.parametrize("kind", ["layer", "rms"])
def test_norm_gradient_is_the_forward_passs(kind):
    """central differences of the 64-bit forward pass along random directions of x, w and b: step h, error h^2 times the third
    derivative, which is below 1e3 for rows of unit variance; taken as 1e-6 for h = 1e-5 beside the gradients' own 1e-5"""
    dev = torch.device("cuda:0")
    g = gen(5)
    m, n = 6, 96
    x, w, b, dy = torch.randn(m, n, generator=g).double(), torch.rand(n, generator=g).double(), torch.randn(n, generator=g).double(), torch.randn(m, n, generator=g).double()
    x, w, b, dy = (t.float().double() for t in (x, w, b, dy))
    out, mean, rstd = torch.empty(m, n, device=dev), torch.empty(m, device=dev), torch.empty(m, device=dev)
    on = lambda t: t.float().to(dev)  # noqa: E731
    mm16.norm(on(x), on(w), out, b=on(b), eps=EPS, kind=kind, mean=mean, rstd=rstd)
    dx, dw, db = torch.empty(m, n, device=dev), torch.empty(n, device=dev), torch.empty(n, device=dev)
    ws = torch.empty(mm16.norm_bwd_ws_bytes(m, n), dtype=torch.uint8, device=dev)
    mm16.norm_bwd(on(x), on(dy), on(w), rstd, dx, mean=mean if kind == "layer" else None, kind=kind, dw=dw, db=db if kind == "layer" else None, ws=ws)
    loss = lambda x, w, b: float((norm64(x, w, b, kind == "layer")[0] * dy).sum())  # noqa: E731
    for i in range(8):
        vx, vw, vb = torch.randn(m, n, generator=g).double(), torch.randn(n, generator=g).double(), torch.randn(n, generator=g).double()
        if kind == "rms":
            vb.zero_()
        h = 1e-5
        diff = (loss(x + h * vx, w + h * vw, b + h * vb) - loss(x - h * vx, w - h * vw, b - h * vb)) / (2 * h)
        terms = (dx.double().cpu() * vx).sum() + (dw.double().cpu() * vw).sum() + ((db.double().cpu() * vb).sum() if kind == "layer" else 0)
        size = (dx.double().cpu() * vx).abs().sum() + (dw.double().cpu() * vw).abs().sum() + (db.double().cpu() * vb).abs().sum() * (kind == "layer")
        assert abs(float(terms) - diff) <= 1e-5 * float(size) + 1e-6, (kind, i, float(terms), diff)


def test_norms_captured_replayed_and_on_another_stream():
    """a step of norm and norm_bwd in a graph and on a stream of its own: the eager bits, replay after replay"""
    dev = torch.device("cuda:0")
    m, n = 300, 2048
    x = torch.empty(m, n, device=dev)
    d, dy = torch.randn(m, n, generator=gen(1)).to(dev), torch.randn(m, n, generator=gen(2)).to(dev).to(BF)
    w = torch.rand(n, generator=gen(3)).to(dev)
    ws = torch.empty(mm16.norm_bwd_ws_bytes(m, n), dtype=torch.uint8, device=dev)

    def buffers():
        return dict(y=torch.empty(m, n, device=dev, dtype=BF), total=torch.empty(m, n, device=dev), mean=torch.empty(m, device=dev), rstd=torch.empty(m, device=dev),
                    dx=torch.empty(m, n, device=dev), dw=torch.empty(n, device=dev), db=torch.empty(n, device=dev))

    def step(o, stream=None):
        mm16.norm(x, w, o["y"], b=w, add=d, total=o["total"], mean=o["mean"], rstd=o["rstd"], stream=stream)
        mm16.norm_bwd(o["total"], dy, w, o["rstd"], o["dx"], mean=o["mean"], resid=d, dw=o["dw"], db=o["db"], ws=ws, stream=stream)
    a, b, c = buffers(), buffers(), buffers()
    x.copy_(torch.randn(m, n, generator=gen(9)))
    step(b)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step(b)
    for seed in range(4):
        x.copy_(torch.randn(m, n, generator=gen(10 + seed)))
        step(a)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        s = torch.cuda.Stream()
        step(c, s)
        s.synchronize()
        for k in a:
            assert torch.equal(a[k], b[k]) and torch.equal(a[k], c[k]), (seed, k)


@pytest.mark.parametrize("n", [600, 767, 768, 769, 1025, 1200, 1536, 1537, 2049, 2304, 2560, 2561, 5001, 6144, 6145, 9001, 12288, 12289])
def test_norm_widths_between_the_powers_of_two(n):
    """rows that their own number of threads takes, few and many of them, forward and backward"""
    dev = torch.device("cuda:0")
    for i, (m, xt) in enumerate(((3, F32), (37, BF), (1700 if n < 4000 else 300, FP), (1700 if n < 4000 else 300, F32))):
        pad, offset = ((0, 0), (3, 1), (0, 0), (1, 2))[i]
        check_norm(("layer", "rms")[i % 2], m, n, xt, (BF, F32, FP, F32)[i], i != 1, i % 2 == 0, dev, n + i, pad, offset)
        check_bwd(("rms", "layer", "layer", "layer")[i], m, n, xt, (F32, BF, F32, FP)[i], i != 0, dev, n + 7 * i, pad, offset)


@pytest.mark.parametrize("n", [1, 5, 9, 505, 506, 512, 1001, 1017, 1018, 1024, 1530, 2041, 2042, 2047, 2560, 4089, 4095, 4096, 6143, 8185, 8186, 8192])
def test_norm_rows_off_their_boundaries(n):
    """rows whose starts go through every place between two 16-byte boundaries, other matrices' rows at other places, and lengths around
    those whose threads have no room for it; blocks of one and of several turns"""
    dev = torch.device("cuda:0")
    g = gen(n)
    for i, (m, xt, yt, kind) in enumerate(((9, BF, F32, "layer"), (25, FP, FP, "rms"), (18, F32, BF, "layer"), (1601 if n < 2100 else 1030, BF, BF, "layer"))):
        check_norm(kind, m, n, xt, yt, i != 2, kind == "layer", dev, n + i, 1 + 2 * i, i, out32=i == 0)
        check_bwd(kind, m, n, xt, yt, i != 1, dev, n + 9 * i, 1 + 2 * i, 3 - i, accumulate=i == 3)
        # each matrix with a place of its own
        x, d, w = rows(g, m, n, xt), rows(g, m, n, xt), torch.rand(n, generator=g).double()
        w = w.float().double()
        outs = [torch.full((m, n + p), 7.0, dtype=xt, device=dev)[:, :n] for p in (3, 6)]
        mm16.norm(put(x, xt, dev, 1, 0), w.float().to(dev), outs[1], kind=kind, add=put(d, xt, dev, 2, 1), total=outs[0])
        same(outs[0], (x + d).to(F32).to(xt).double(), f"total {m}x{n}")
        s = outs[0].double().cpu()
        y, mu, r = norm64(s, w, None, kind == "layer")
        mu_err = (depth(n) + 2) * u * s.abs().mean(1, keepdim=True) if kind == "layer" else torch.zeros_like(mu)
        r_rel = 0.5 * ((depth(n) + 4) * u + mu_err ** 2 * r * r) + 3 * u
        within(outs[1], y, ((s - mu) * r * w).abs() * (r_rel + 4 * u) + mu_err * r * w.abs() + 2 * u * y.abs(), f"{kind} {m}x{n} {xt}")
        assert (outs[0]._base[:, n:] == 7.0).all() and (outs[1]._base[:, n:] == 7.0).all()


@pytest.mark.parametrize("dt", [F32, BF])
@pytest.mark.parametrize("n", [9, 1001, 2047, 4093, 6001, 9001, 14001])
def test_norm_in_place_with_pieces_that_overlap(n, dt):
    """rows whose last piece starts inside the one before, in the place of every matrix that may be: bit for bit as in places of
    their own, whichever thread comes first"""
    dev = torch.device("cuda:0")
    g = gen(n)
    for m in (40, 1100) if n < 5000 else (40, 300):
        for kind in ("layer", "rms"):
            x, d = torch.randn(m, n, generator=g).to(dt).to(dev), torch.randn(m, n, generator=g).to(dt).to(dev)
            w = torch.rand(n, generator=g).to(dev)
            total, out, mean, rstd = torch.empty_like(x), torch.empty_like(x), torch.empty(m, device=dev), torch.empty(m, device=dev)
            mm16.norm(x, w, out, kind=kind, add=d, total=total, mean=mean, rstd=rstd)
            for place in ("x", "add"):
                a, b, o = x.clone(), d.clone(), torch.empty_like(x)
                mm16.norm(a, w, o, kind=kind, add=b, total=a if place == "x" else b)
                assert torch.equal(o, out) and torch.equal(a if place == "x" else b, total), (m, n, kind, place)
            a = total.clone()
            mm16.norm(a, w, a, kind=kind)
            assert torch.equal(a, out)
            dy, e = torch.randn(m, n, generator=g).to(dt).to(dev), torch.randn(m, n, generator=g).to(dt).to(dev)
            ws = torch.empty(mm16.norm_bwd_ws_bytes(m, n), dtype=torch.uint8, device=dev)

            def back(px, py, pe, pd):
                dw, db = torch.empty(n, device=dev), torch.empty(n, device=dev) if kind == "layer" else None
                mm16.norm_bwd(px, py, w, rstd, pd, mean=mean, kind=kind, resid=pe, dw=dw, db=db, ws=ws)
                return pd, dw, db if db is not None else dw

            want = back(total, dy, e, torch.empty_like(x))
            for place in range(3):
                p = [total.clone(), dy.clone(), e.clone()]
                got = back(*p, p[place])
                assert all(torch.equal(s, t) for s, t in zip(got, want)), (m, n, kind, dt, place)
