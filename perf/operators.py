"""Performance cases of the 16-bit matrix products: linear layers with bias, activation and residual, products grouped by
expert, their gradients and the SwiGLU gradient between them, as a serving step or a training step calls them.

A case's `op`:
  linear       out = act(x W^T + b) (+ resid);  m rows, n outputs, k inputs; `save` keeps the pre-activation z as well
  linear_bwd   dx = dz W,  dW = dz^T x,  db = sum of dz over the rows
  gate_up      h[p] = silu(Wg_e x_t) * (Wu_e x_t) for the pairs p = t topk + j of token t with expert e; `save` keeps both products
  down         y[p] = w[p] Wd_e h[p]
  moe_bwd      the products of a training step's backward pass: dh[p] = dy_t Wd_e,  dx[p] = dg[p] Wg_e + du[p] Wu_e and the three
               weights' gradients, each the sum over the expert's pairs
  glu_bwd      gradient of w[p] silu(g) u: dg, du, w h (the down weights' operand) and the routing weights' gradient
`type` is the 16-bit type of inputs and weights; `f32` says that outputs (of linear and down: the residual stream; of the
backward passes: the weights' gradients) are float32.  d, E, topk, ff: d_model, experts, experts a token, expert width.
`zipf`: tokens per expert follow Zipf(zipf).  `by_ids`: no grouping, each pair by its expert id (single tokens).
"""
import math

import torch

own = False
DEV = "cuda"
TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16}


def _linear(op, type_, m, n, k, act="none", bias=False, resid=False, f32=False, save=False):
    return dict(op=op, type=type_, m=m, n=n, k=k, act=act, bias=bias, resid=resid, f32=f32, save=save)


def _moe(op, type_, d, E, topk, ff, rows, zipf=0.0, by_ids=False, f32=False, save=False):
    return dict(op=op, type=type_, d=d, E=E, topk=topk, ff=ff, rows=rows, zipf=zipf, by_ids=by_ids, f32=f32, save=save)


def listed():
    return [
        # the attention output projection of one generated token, added into the fp32 residual stream: launch latency
        dict(_linear("linear", "bf16", 1, 2048, 2048, bias=True, resid=True, f32=True), name="linear 1 row"),
        # a ragged prompt through a layer of odd width, the pre-activation kept for the backward pass
        dict(_linear("linear", "fp16", 509, 1000, 2048, act="gelu", bias=True, save=True), name="linear 509 rows"),
        # a batch of long sequences through a wide feed-forward matrix
        dict(_linear("linear", "bf16", 8192, 7168, 4096, act="silu"), name="linear 8192 rows"),
        # the backward pass of the ragged layer
        dict(_linear("linear_bwd", "fp16", 509, 1000, 2048), name="linear backward 509 rows"),
        # the backward pass of a training batch, weight gradients in float32
        dict(_linear("linear_bwd", "bf16", 8192, 4096, 4096, f32=True), name="linear backward 8192 rows"),
        # one generated token through the experts (d 2048, 128 experts, top-8, ff 768)
        dict(_moe("gate_up", "bf16", 2048, 128, 8, 768, 1, by_ids=True), name="gate/up 1 token"),
        # a 512-token prompt with skewed routing: the weights of nearly every expert
        dict(_moe("gate_up", "bf16", 2048, 128, 8, 768, 512, zipf=1.1), name="gate/up 512 tokens"),
        # a training batch: every expert has about a thousand rows, gate and up kept
        dict(_moe("gate_up", "fp16", 2048, 64, 8, 1024, 8192, save=True), name="gate/up 8192 tokens"),
        # a ragged prompt through a wide layer, fp32 rows for the combine: the largest weights
        dict(_moe("down", "bf16", 4096, 288, 8, 1536, 1000, zipf=1.1, f32=True), name="down 1000 tokens"),
        # the backward products of a training batch
        dict(_moe("moe_bwd", "bf16", 2048, 64, 8, 1024, 2048), name="experts backward 2048 tokens"),
        # the activation's gradient for a few short sequences, and for the training batch
        dict(_moe("glu_bwd", "fp16", 2048, 128, 8, 768, 37), name="glu backward 37 tokens"),
        dict(_moe("glu_bwd", "bf16", 2048, 64, 8, 1024, 8192), name="glu backward 8192 tokens"),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


# expert layers: (d, most experts, top-k, ff, most rows), sizes as the listed ones'
_LAYERS = [(2048, 128, 8, 768, 4096), (4096, 288, 8, 1536, 1000), (2048, 64, 8, 1024, 8192), (2048, 512, 10, 512, 2048), (1024, 16, 2, 1000, 8192)]


def draw(rng):
    op = rng.choice(["linear", "linear", "linear_bwd", "gate_up", "gate_up", "down", "moe_bwd", "glu_bwd"])
    type_ = rng.choice(["bf16", "fp16"])
    if op in ("linear", "linear_bwd"):
        m = _log(rng, 1, 8192) if op == "linear" else _log(rng, 16, 8192)
        n, k = (_log(rng, 256, 7168) if rng.random() < 0.3 else 8 * _log(rng, 32, 896) for _ in range(2))
        if op == "linear_bwd":
            return _linear(op, type_, m, min(n, 4096), min(k, 4096), f32=rng.random() < 0.5)
        return _linear(op, type_, m, n, min(k, 4096), act=rng.choice(["none", "relu", "silu", "gelu", "gelu_tanh"]), bias=rng.random() < 0.5,
                       resid=rng.random() < 0.5, f32=rng.random() < 0.3, save=rng.random() < 0.3)
    d, E, topk, ff, most = rng.choice([v for v in _LAYERS if op != "moe_bwd" or v[1] <= 128])   # three weights and their gradients
    if op == "gate_up":
        E = min(E, 128 if d == 4096 else 512)   # two weights
    E = max(topk, E - rng.choice([0, 0, 1, 5]))
    if op == "gate_up" and rng.random() < 0.3:
        return _moe(op, type_, d, E, topk, ff, rng.choice([1, 1, 2, 4]), by_ids=True)
    rows = _log(rng, 2 if op != "moe_bwd" else 32, most if op != "moe_bwd" else min(most, 2048))
    return _moe(op, type_, d, E, topk, ff, rows, zipf=rng.choice([0.0, 0.0, 1.1]), f32=op in ("down", "moe_bwd") and rng.random() < 0.5,
                save=op == "gate_up" and rng.random() < 0.3)


# ------------------------------------------------------------------ what a program has in hand

def _randn(g, *shape, dtype, scale=1.0):
    return torch.randn(*shape, generator=g, device=DEV, dtype=dtype).mul_(scale)


def prepare(case, seed):
    c = case
    g = torch.Generator(device=DEV)
    g.manual_seed(9176 * int(seed) + 77)
    T = TYPES[c["type"]]
    s = {"c": c}
    if "m" in c:
        m, n, k = c["m"], c["n"], c["k"]
        s["W"] = _randn(g, n, k, dtype=T, scale=k ** -0.5)
        # rows of uneven norms, as hidden rows have
        s["x"] = _randn(g, m, k, dtype=T) * torch.exp(0.5 * torch.randn(m, 1, generator=g, device=DEV)).to(T)
        if c["op"] == "linear_bwd":
            s["dz"] = _randn(g, m, n, dtype=T, scale=0.1)
            return s
        s["bias"] = _randn(g, n, dtype=torch.float32, scale=0.5) if c["bias"] else None
        s["resid"] = _randn(g, m, n, dtype=torch.float32 if c["f32"] else T) if c["resid"] else None
        return s
    d, E, topk, ff, rows = c["d"], c["E"], c["topk"], c["ff"], c["rows"]
    P = rows * topk
    if c["op"] == "glu_bwd":
        s["g"], s["u"] = _randn(g, P, ff, dtype=T), _randn(g, P, ff, dtype=T)
        s["dh"] = _randn(g, P, ff, dtype=T, scale=0.1)
        s["wts"] = torch.rand(P, generator=g, device=DEV) / topk
        return s
    # the routing: topk distinct experts a token, skewed where asked, and its grouping as the bucketing kernel leaves it
    score = torch.rand(rows, E, generator=g, device=DEV).clamp_min_(1e-9).log_().neg_().log_().neg_()
    if c["zipf"]:
        score -= c["zipf"] * torch.log(torch.arange(1, E + 1, device=DEV, dtype=torch.float32))
    ids = score.topk(topk, dim=1).indices.reshape(-1)
    s["ids"] = ids.to(torch.int32)
    s["slot"] = torch.arange(E, dtype=torch.int32, device=DEV)
    s["wts"] = torch.rand(P, generator=g, device=DEV) / topk
    if not c["by_ids"]:
        order = torch.argsort(ids, stable=True)
        cnt = torch.bincount(ids, minlength=E)
        start = torch.cumsum(cnt, 0) - cnt
        act = torch.nonzero(cnt).reshape(-1)
        s["order"] = order.to(torch.int32)
        s["order_n"] = torch.tensor([P, act.numel()], dtype=torch.int32, device=DEV)
        egrp = torch.zeros(E, 3, dtype=torch.int32, device=DEV)
        egrp[:act.numel()] = torch.stack([act, start[act], cnt[act]], 1).to(torch.int32)
        s["egrp"] = egrp.reshape(-1)
        s["max_active"] = min(E, P)
        # the groups cut into blocks of `blk` pairs, for batched products: the blocks' experts, and their pairs (P: none)
        blk = max(16, 1 << max(0, math.ceil(math.log2(max(1.0, P / E)))))
        nb = (cnt + blk - 1) // blk
        be = torch.repeat_interleave(torch.arange(E, device=DEV), nb)
        first = torch.cumsum(nb, 0) - nb
        at = (torch.arange(be.numel(), device=DEV) - first[be])[:, None] * blk + torch.arange(blk, device=DEV)[None]
        inside = at < cnt[be][:, None]
        pos = torch.where(inside, start[be][:, None] + at, torch.zeros_like(at))
        s["blk_e"], s["blk_p"] = be, torch.where(inside, order[pos], torch.full_like(at, P))
    if c["op"] != "down":
        s["gate"] = _randn(g, E, ff, d, dtype=T, scale=d ** -0.5)
        s["up"] = _randn(g, E, ff, d, dtype=T, scale=d ** -0.5)
        s["x"] = _randn(g, rows, d, dtype=T) * torch.exp(0.5 * torch.randn(rows, 1, generator=g, device=DEV)).to(T)
    if c["op"] != "gate_up":
        s["down"] = _randn(g, E, d, ff, dtype=T, scale=ff ** -0.5)
    if c["op"] == "down":
        s["h"] = _randn(g, P, ff, dtype=T, scale=0.5)
    if c["op"] == "moe_bwd":
        s["dy"] = _randn(g, rows, d, dtype=T, scale=0.1)
        s["dg"], s["du"] = _randn(g, P, ff, dtype=T, scale=0.1), _randn(g, P, ff, dtype=T, scale=0.1)
        s["hw"] = _randn(g, P, ff, dtype=T, scale=0.1)
    return s


# ------------------------------------------------------------------ the framework's calls

def _dev(s):
    """the layer descriptor that a program keeps beside its weights"""
    if "dev" not in s:
        from hyper_amd import mm16
        s["dev"] = mm16.Moe16Dev(s.get("gate"), s.get("up"), s.get("down"), s["slot"])
    return s["dev"]


def _run_own(s):
    from hyper_amd import mm16
    c = s["c"]
    T = TYPES[c["type"]]
    new = lambda *shape, dtype=T: torch.empty(*shape, dtype=dtype, device=DEV)  # noqa: E731
    F = torch.float32 if c["f32"] else T
    if c["op"] == "linear":
        out = new(c["m"], c["n"], dtype=F)
        z = new(c["m"], c["n"]) if c["save"] else None
        mm16.linear(s["W"], s["x"], out, bias=s["bias"], act=c["act"], resid=s["resid"], z=z)
        return {"out": out, "z": z} if c["save"] else {"out": out}
    if c["op"] == "linear_bwd":
        dx, dW, db = new(c["m"], c["k"]), new(c["n"], c["k"], dtype=F), new(c["n"], dtype=torch.float32)
        ws = new(mm16.linear_dw_ws_bytes(c["m"], c["n"], c["k"]), dtype=torch.uint8)
        mm16.linear_dx(s["W"], s["dz"], dx)
        mm16.linear_dw(s["dz"], s["x"], dW, db=db, ws=ws)
        return {"dx": dx, "dW": dW, "db": db}
    d, E, topk, ff, rows = c["d"], c["E"], c["topk"], c["ff"], c["rows"]
    P = rows * topk
    if c["op"] == "glu_bwd":
        dg, du, hw, dwts = new(P, ff), new(P, ff), new(P, ff), new(P, dtype=torch.float32)
        mm16.swiglu_bwd(s["g"], s["u"], s["dh"], s["wts"], dg, du, hw, dwts)
        return {"dg": dg, "du": du, "hw": hw, "dwts": dwts}
    m = _dev(s)
    if c["op"] == "gate_up":
        h = new(P, ff)
        gu = {"g": new(P, ff), "u": new(P, ff)} if c["save"] else {}
        if c["by_ids"]:
            mm16.moe16_gate_up(m, s["x"], topk, P, h, ids=s["ids"], **gu)
        else:
            mm16.moe16_gate_up(m, s["x"], topk, P, h, order=s["order"], order_n=s["order_n"], egrp=s["egrp"], max_active=s["max_active"], **gu)
        return {"h": h, **gu}
    grp = (s["order"], s["order_n"], s["egrp"], s["max_active"])
    if c["op"] == "down":
        y = new(P, d, dtype=F)
        mm16.moe16_down(m, s["h"], P, y, wts=s["wts"], order=grp[0], order_n=grp[1], egrp=grp[2], max_active=grp[3])
        return {"y": y}
    dh, dx = new(P, ff), new(P, d)
    dwg, dwu, dwd = new(E, ff, d, dtype=F), new(E, ff, d, dtype=F), new(E, d, ff, dtype=F)
    mm16.moe16_down_dx(m, s["dy"], topk, P, *grp, dh)
    mm16.moe16_gate_up_dx(m, s["dg"], s["du"], P, *grp, dx)
    mm16.moe16_dw(m, s["dg"], 1, s["x"], topk, P, *grp, dwg)
    mm16.moe16_dw(m, s["du"], 1, s["x"], topk, P, *grp, dwu)
    mm16.moe16_dw(m, s["dy"], topk, s["hw"], 1, P, *grp, dwd)
    return {"dh": dh, "dx": dx, "dwg": dwg, "dwu": dwu, "dwd": dwd}


# ------------------------------------------------------------------ the plain form

def _act(name, z):
    if name == "relu":
        return z.clamp_min(0)
    if name == "silu":
        return z * torch.sigmoid(z)
    if name == "gelu":
        return 0.5 * z * torch.erfc(z * -(0.5 ** 0.5))
    if name == "gelu_tanh":   # 0.5 z (1 + tanh(a)) = z sigmoid(2 a)
        return z * torch.sigmoid(2 * math.sqrt(2 / math.pi) * (z + 0.044715 * z * z * z))
    return z


def _rows(t, at):
    """fp32 rows of t, with rows of zeros where `at` points behind its end"""
    return torch.cat([t.float(), torch.zeros_like(t[:1], dtype=torch.float32)])[at]


def _back(blocks, blk_p, P):
    """the blocks' rows at their pairs"""
    out = blocks.new_zeros(P + 1, blocks.shape[-1])
    out[blk_p.reshape(-1)] = blocks.reshape(-1, blocks.shape[-1])
    return out[:P]


def _per_expert(blocks, blk_e, E):
    """the blocks' matrices summed by expert"""
    return blocks.new_zeros(E, *blocks.shape[1:]).index_add_(0, blk_e, blocks)


def run(state):
    s = state
    if own:
        return _run_own(s)
    c = s["c"]
    T = TYPES[c["type"]]
    F = torch.float32 if c["f32"] else T
    if c["op"] == "linear":
        z = s["x"].float() @ s["W"].float().t()
        if s["bias"] is not None:
            z = z + s["bias"]
        out = _act(c["act"], z)
        if s["resid"] is not None:
            out = out + s["resid"].float()
        return {"out": out.to(F), "z": z.to(T)} if c["save"] else {"out": out.to(F)}
    if c["op"] == "linear_bwd":
        dz = s["dz"].float()
        return {"dx": (dz @ s["W"].float()).to(T), "dW": (dz.t() @ s["x"].float()).to(F), "db": dz.sum(0)}
    d, E, topk, rows = c["d"], c["E"], c["topk"], c["rows"]
    P = rows * topk
    if c["op"] == "glu_bwd":
        g, u, dh, w = s["g"].float(), s["u"].float(), s["dh"].float(), s["wts"][:, None]
        sig = torch.sigmoid(g)
        silu = g * sig
        return {"dg": (w * dh * u * (sig + silu * (1 - sig))).to(T), "du": (w * dh * silu).to(T), "hw": (w * silu * u).to(T),
                "dwts": (dh * silu * u).sum(1)}
    if c["by_ids"]:
        x = s["x"].float().repeat_interleave(topk, 0)[:, :, None]
        ids = s["ids"].long()
        g, u = (torch.bmm(s[n][ids].float(), x)[:, :, 0] for n in ("gate", "up"))
        h = (g * torch.sigmoid(g) * u).to(T)
        return {"h": h, "g": g.to(T), "u": u.to(T)} if c["save"] else {"h": h}
    be, bp = s["blk_e"], s["blk_p"]
    tok = torch.where(bp < P, bp // topk, torch.full_like(bp, rows))
    if c["op"] == "gate_up":
        x = _rows(s["x"], tok)
        g, u = (_back(torch.bmm(x, s[n][be].float().transpose(1, 2)), bp, P) for n in ("gate", "up"))
        h = (g * torch.sigmoid(g) * u).to(T)
        return {"h": h, "g": g.to(T), "u": u.to(T)} if c["save"] else {"h": h}
    if c["op"] == "down":
        y = _back(torch.bmm(_rows(s["h"], bp), s["down"][be].float().transpose(1, 2)), bp, P)
        return {"y": (y * s["wts"][:, None]).to(F)}
    dy, dg, du, hw, x = _rows(s["dy"], tok), _rows(s["dg"], bp), _rows(s["du"], bp), _rows(s["hw"], bp), _rows(s["x"], tok)
    dh = _back(torch.bmm(dy, s["down"][be].float()), bp, P)
    dx = _back(torch.bmm(dg, s["gate"][be].float()) + torch.bmm(du, s["up"][be].float()), bp, P)
    dwg, dwu, dwd = (_per_expert(torch.bmm(a.transpose(1, 2).contiguous(), b), be, E).to(F) for a, b in ((dg, x), (du, x), (dy, hw)))
    return {"dh": dh.to(T), "dx": dx.to(T), "dwg": dwg, "dwu": dwu, "dwd": dwd}


# ------------------------------------------------------------------ what a pass cannot do without

def _touched(c):
    """expected distinct experts of a call: each is missed by a row with probability 1 - (its share of topk)"""
    E, k, R = c["E"], c["topk"], c["rows"]
    p = [1.0 / (r + 1) ** c["zipf"] for r in range(E)]
    return sum(1 - (1 - min(1.0, k * v / sum(p))) ** R for v in p)


def work(case):
    c = case
    if "m" in c:
        m, n, k = c["m"], c["n"], c["k"]
        if c["op"] == "linear_bwd":
            return {"bytes": 2.0 * (2 * m * k + n * k + m * n) + n * k * (4 if c["f32"] else 2) + 4 * n, "flops": 4.0 * m * n * k}
        o = 4 if c["f32"] else 2
        return {"bytes": 2.0 * (m * k + n * k) + m * n * (o * (2 if c["resid"] else 1) + (2 if c["save"] else 0)) + (4 * n if c["bias"] else 0),
                "flops": 2.0 * m * n * k}
    d, E, topk, ff, rows = c["d"], c["E"], c["topk"], c["ff"], c["rows"]
    P = rows * topk
    if c["op"] == "glu_bwd":
        return {"bytes": 12.0 * P * ff + 8 * P, "flops": 20.0 * P * ff}
    mat = 2.0 * _touched(c) * ff * d
    if c["op"] == "gate_up":
        return {"bytes": 2 * mat + 2.0 * rows * d + 2.0 * P * ff * (3 if c["save"] else 1), "flops": 4.0 * P * ff * d}
    o = 4 if c["f32"] else 2
    if c["op"] == "down":
        return {"bytes": mat + 2.0 * P * ff + o * P * d, "flops": 2.0 * P * ff * d}
    return {"bytes": 3 * mat + 3.0 * o * E * ff * d + 2.0 * (2 * rows * d + 4 * P * ff + P * d), "flops": 12.0 * P * ff * d}


# ------------------------------------------------------------------ the same in 64 bits

def exact(case, seed):
    c, s = case, prepare(case, seed)
    D = lambda t: t.double()  # noqa: E731
    if c["op"] == "linear":
        z = torch.addmm(D(s["bias"]), D(s["x"]), D(s["W"]).t()) if c["bias"] else torch.mm(D(s["x"]), D(s["W"]).t())
        a = c["act"]
        if a == "none":
            out = z
        elif a == "relu":
            out = torch.where(z > 0, z, torch.zeros_like(z))
        elif a == "silu":
            out = z / (1 + torch.exp(-z))
        elif a == "gelu":
            out = z * 0.5 * (1 + torch.erf(z / math.sqrt(2)))
        else:
            out = z * 0.5 * (1 + torch.tanh(math.sqrt(2 / math.pi) * (z + 0.044715 * z ** 3)))
        out = out + D(s["resid"]) if c["resid"] else out
        return {"out": out, "z": z} if c["save"] else {"out": out}
    if c["op"] == "linear_bwd":
        return {"dx": torch.mm(D(s["dz"]), D(s["W"])), "dW": torch.mm(D(s["dz"]).t(), D(s["x"])), "db": D(s["dz"]).sum(0)}
    E, topk, ff, d = c["E"], c["topk"], c["ff"], c["d"]
    P = c["rows"] * topk
    new = lambda *shape: torch.zeros(*shape, dtype=torch.float64, device=DEV)  # noqa: E731
    if c["op"] == "glu_bwd":
        g, u, dh, w = D(s["g"]), D(s["u"]), D(s["dh"]), D(s["wts"])[:, None]
        e = 1 + torch.exp(-g)
        h = g * u / e
        return {"dg": w * dh * u * (1 / e + g * (e - 1) / e ** 2), "du": w * dh * g / e, "hw": w * h, "dwts": (dh * h).sum(1)}
    ids = s["ids"].long()
    pairs = [torch.nonzero(ids == e).reshape(-1) for e in range(E)]
    if c["op"] == "gate_up":
        out = {n: new(P, ff) for n in ("h", "g", "u")}
        for e, p in enumerate(pairs):
            x = D(s["x"][p // topk])
            g, u = x @ D(s["gate"][e]).t(), x @ D(s["up"][e]).t()
            out["h"][p], out["g"][p], out["u"][p] = g / (1 + torch.exp(-g)) * u, g, u
        return out if c["save"] else {"h": out["h"]}
    if c["op"] == "down":
        y = new(P, d)
        for e, p in enumerate(pairs):
            y[p] = (D(s["h"][p]) @ D(s["down"][e]).t()) * D(s["wts"][p])[:, None]
        return {"y": y}
    out = {"dh": new(P, ff), "dx": new(P, d), "dwg": new(E, ff, d), "dwu": new(E, ff, d), "dwd": new(E, d, ff)}
    for e, p in enumerate(pairs):
        x, dy, dg, du, hw = D(s["x"][p // topk]), D(s["dy"][p // topk]), D(s["dg"][p]), D(s["du"][p]), D(s["hw"][p])
        out["dh"][p] = dy @ D(s["down"][e])
        out["dx"][p] = dg @ D(s["gate"][e]) + du @ D(s["up"][e])
        out["dwg"][e], out["dwu"][e], out["dwd"][e] = dg.t() @ x, du.t() @ x, dy.t() @ hw
    return out
