"""Performance cases of the operators around the 16-bit products of a block: norms, routing with groups, low-rank adapters, and
the gradients of the first two, as a serving step or a training step calls them.

A case's `op`:
  norm        y = (s - mean) rstd w + b of rows s = x + add ("layer"; "rms": no mean, no b); `add`: s is written as well;
              `x32`: x, add and s are float32 (the residual stream), else of the 16-bit type; y is of the 16-bit type; the rows'
              statistics are kept for the backward pass
  norm_bwd    dx (+ the gradient that passes by on the residual stream), dw, db from dy of the 16-bit type
  route       scores (softmax or sigmoid) of E experts, a selection bias, the best `top_group` of `n_group` groups by the sum
              of their `best` best, the k best experts in them, weights renormalised and scaled; `coarse`: logits with many ties
  route_bwd   gradient of the weights with respect to the logits; `d32`: in float32, else in bfloat16, for the router's products
  lora        out = base + scale_a B_a A_a x for rows of many requests, each with its adapter a (or none); rank r, k inputs,
              n outputs; `lengths`: "one" (a generated token a request), "ragged" (prompts of different lengths)
"""
import math

import torch

own = False
DEV = "cuda"
TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16}


def _norm(op, type_, kind, m, n, x32=True, add=False):
    return dict(op=op, type=type_, kind=kind, m=m, n=n, x32=x32, add=add)


def _route(op, score, nt, E, k, n_group=1, top_group=1, best=1, bias=False, renorm=True, scale=1.0, coarse=False, d32=True):
    return dict(op=op, score=score, nt=nt, E=E, k=k, n_group=n_group, top_group=top_group, best=best, bias=bias, renorm=renorm,
                scale=scale, coarse=coarse, d32=d32)


def _lora(type_, m, k, n, r, adapters, requests, lengths, f32=False):
    return dict(op="lora", type=type_, m=m, k=k, n=n, r=r, adapters=adapters, requests=requests, lengths=lengths, f32=f32)


def listed():
    return [
        # the norm in front of an expert layer for one generated token, the attention's output added on the way: latency
        dict(_norm("norm", "bf16", "rms", 1, 2048, add=True), name="norm 1 row"),
        # a ragged prompt through a layer norm of odd width, 16-bit residual stream
        dict(_norm("norm", "fp16", "layer", 509, 1001, x32=False), name="norm 509 rows"),
        # a training batch in front of a wide layer, fp32 residual stream
        dict(_norm("norm", "bf16", "rms", 8192, 4096, add=True), name="norm 8192 rows"),
        # the backward pass of the ragged prompt and of the training batch
        dict(_norm("norm_bwd", "fp16", "layer", 509, 1001, x32=False), name="norm backward 509 rows"),
        dict(_norm("norm_bwd", "bf16", "rms", 8192, 4096, add=True), name="norm backward 8192 rows"),
        # one generated token: sigmoid scores, a balance bias, half of the groups
        dict(_route("route", "sigmoid", 1, 384, 6, 8, 4, 2, bias=True, scale=2.5), name="route 1 token"),
        # a 512-token prompt, softmax scores rounded to 16 bits before the router, groups by their best expert
        dict(_route("route", "softmax", 512, 128, 8, 8, 3, 1, coarse=True), name="route 512 tokens"),
        # a training batch: sigmoid scores, bias, groups
        dict(_route("route", "sigmoid", 8192, 256, 8, 8, 4, 2, bias=True, scale=2.5), name="route 8192 tokens"),
        # the router's gradient of a few short sequences (weights not renormalised: every expert's logit gets one), and of a batch
        dict(_route("route_bwd", "softmax", 37, 128, 8, renorm=False), name="route backward 37 tokens"),
        dict(_route("route_bwd", "sigmoid", 8192, 256, 8, 8, 4, 2, bias=True, scale=2.5, d32=False), name="route backward 8192 tokens"),
        # one generated token each of 16 requests with their own adapters beside an attention projection
        dict(_lora("bf16", 16, 4096, 4096, 16, 64, 16, "one"), name="adapters 16 rows"),
        # prompts of 24 requests beside a wide feed-forward matrix
        dict(_lora("bf16", 4096, 4096, 7168, 64, 32, 24, "ragged"), name="adapters 4096 rows"),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


# experts and group counts that divide them
_EXPERTS = [(16, (1, 2, 4)), (60, (1, 3, 6)), (128, (1, 4, 8)), (160, (1, 8)), (256, (1, 8, 16)), (288, (1, 8)), (384, (1, 8)), (512, (1, 8, 16))]


def draw(rng):
    op = rng.choice(["norm", "norm", "norm_bwd", "norm_bwd", "route", "route", "route_bwd", "lora", "lora", "lora"])
    type_ = rng.choice(["bf16", "fp16"])
    if op in ("norm", "norm_bwd"):
        n = _log(rng, 64, 8192) if rng.random() < 0.4 else 8 * _log(rng, 8, 1024)
        m = _log(rng, 1 if op == "norm" else 2, min(16384, 8192 * 4096 // n))
        return _norm(op, type_, rng.choice(["layer", "rms"]), m, n, x32=rng.random() < 0.6, add=rng.random() < 0.5)
    if op in ("route", "route_bwd"):
        E, groups = rng.choice(_EXPERTS)
        n_group = rng.choice(groups)
        top_group = rng.randint(1, n_group)
        best = rng.choice([1, 2])
        k = rng.randint(1, min(10, E // n_group * top_group))
        return _route(op, rng.choice(["softmax", "sigmoid"]), _log(rng, 1, 8192 * 256 // max(E, 256)), E, k, n_group, top_group, best,
                      bias=rng.random() < 0.6, renorm=k > 1 and rng.random() < 0.7, scale=rng.choice([1.0, 2.5]), coarse=rng.random() < 0.3,
                      d32=rng.random() < 0.5)
    k, n = (_log(rng, 256, 7168) if rng.random() < 0.2 else 8 * _log(rng, 32, 896) for _ in range(2))
    k, r, adapters = min(k, 4096), rng.choice([4, 8, 8, 16, 16, 16, 20, 32, 64]), rng.randint(1, 32)
    if rng.random() < 0.4:
        m = _log(rng, 1, 128)
        return _lora(type_, m, k, n, r, adapters, m, "one", f32=rng.random() < 0.3)
    m = _log(rng, 17, 4096)
    return _lora(type_, m, k, n, r, adapters, rng.randint(1, min(m, 24)), "ragged", f32=False)


# ------------------------------------------------------------------ what a program has in hand

def _randn(g, *shape, dtype, scale=1.0):
    return torch.randn(*shape, generator=g, device=DEV, dtype=dtype).mul_(scale)


def prepare(case, seed):
    c = case
    g = torch.Generator(device=DEV)
    g.manual_seed(7919 * int(seed) + 31)
    s = {"c": c}
    if c["op"] in ("norm", "norm_bwd"):
        m, n, T = c["m"], c["n"], TYPES[c["type"]]
        X = torch.float32 if c["x32"] else T
        # a residual stream: rows of uneven norms, a few columns far larger than the rest, some offset
        col = torch.exp(0.5 * torch.randn(n, generator=g, device=DEV))
        col[torch.randint(0, n, (max(1, n // 512),), generator=g, device=DEV)] *= 20
        x = torch.randn(m, n, generator=g, device=DEV) * col
        x += 0.2
        x *= torch.exp(0.5 * torch.randn(m, 1, generator=g, device=DEV))
        s["x"] = x.to(X)
        s["w"] = 1 + _randn(g, n, dtype=torch.float32, scale=0.2)
        s["b"] = _randn(g, n, dtype=torch.float32, scale=0.1) if c["kind"] == "layer" else None
        if c["op"] == "norm":
            s["add"] = _randn(g, m, n, dtype=X) if c["add"] else None
            return s
        s["dy"] = _randn(g, m, n, dtype=T, scale=0.1)
        s["resid"] = _randn(g, m, n, dtype=X, scale=0.1) if c["add"] else None
        # the statistics as the forward pass leaves them
        d = s["x"].double()
        mean = d.mean(1, keepdim=True) if c["kind"] == "layer" else d.new_zeros(m, 1)
        s["mean"] = mean[:, 0].float()
        s["rstd"] = (((d - mean) ** 2).mean(1) + 1e-5).rsqrt().float()
        return s
    if c["op"] in ("route", "route_bwd"):
        nt, E, k = c["nt"], c["E"], c["k"]
        # router logits: a direction that every token shares, and its own
        logits = _randn(g, nt, E, dtype=torch.float32, scale=1.2) + _randn(g, E, dtype=torch.float32, scale=0.5)
        s["logits"] = logits.to(torch.bfloat16).float() if c["coarse"] else logits
        s["bias"] = _randn(g, E, dtype=torch.float32, scale=0.02) if c["bias"] else None
        if c["op"] == "route_bwd":
            s["ids"] = _choose(c, s)[0].to(torch.int32)
            s["dwts"] = _randn(g, nt, k, dtype=torch.float32, scale=0.1)
        return s
    m, k, n, r, T = c["m"], c["k"], c["n"], c["r"], TYPES[c["type"]]
    F = torch.float32 if c["f32"] else T
    s["A"] = _randn(g, c["adapters"], r, k, dtype=T, scale=k ** -0.5)
    s["B"] = _randn(g, c["adapters"], n, r, dtype=T, scale=r ** -0.5)
    s["scale"] = 0.5 + torch.rand(c["adapters"], generator=g, device=DEV)
    s["x"] = _randn(g, m, k, dtype=T) * torch.exp(0.5 * torch.randn(m, 1, generator=g, device=DEV)).to(T)
    s["base"] = _randn(g, m, n, dtype=F)
    # the requests' adapters, one in eight without; their rows lie one request after the other
    who = torch.randint(0, c["adapters"], (c["requests"],), generator=g, device=DEV)
    who = torch.where(torch.rand(c["requests"], generator=g, device=DEV) < 0.125, torch.full_like(who, -1), who)
    if c["lengths"] == "one":
        s["ids"] = who.to(torch.int32)
    else:
        ends = torch.sort(torch.randperm(m - 1, generator=g, device=DEV)[:c["requests"] - 1] + 1).values if c["requests"] > 1 else who.new_zeros(0)
        s["ids"] = who[torch.searchsorted(ends, torch.arange(m, device=DEV), right=True)].to(torch.int32)
        at = [0, *ends.tolist(), m]   # a program knows its prompts' lengths
        s["prompts"] = list(zip(who.tolist(), at[:-1], at[1:]))
    return s


# ------------------------------------------------------------------ the framework's calls

def _run_own(s):
    from hyper_amd import mm16
    c = s["c"]
    new = lambda *shape, dtype=torch.float32: torch.empty(*shape, dtype=dtype, device=DEV)  # noqa: E731
    if c["op"] == "norm":
        m, n, T = c["m"], c["n"], TYPES[c["type"]]
        y, rstd = new(m, n, dtype=T), new(m)
        mean = new(m) if c["kind"] == "layer" else None
        total = torch.empty_like(s["x"]) if c["add"] else None
        mm16.norm(s["x"], s["w"], y, b=s["b"], eps=1e-5, kind=c["kind"], add=s["add"], total=total, mean=mean, rstd=rstd)
        return {"y": y, "total": total, "mean": mean, "rstd": rstd}
    if c["op"] == "norm_bwd":
        m, n = c["m"], c["n"]
        dx, dw = torch.empty_like(s["x"]), new(n)
        db = new(n) if c["kind"] == "layer" else None
        ws = new(mm16.norm_bwd_ws_bytes(m, n), dtype=torch.uint8)
        mm16.norm_bwd(s["x"], s["dy"], s["w"], s["rstd"], dx, mean=s["mean"] if c["kind"] == "layer" else None, kind=c["kind"], resid=s["resid"],
                      dw=dw, db=db, ws=ws)
        return {"dx": dx, "dw": dw, "db": db}
    if c["op"] == "route":
        ids, wts = new(c["nt"], c["k"], dtype=torch.int32), new(c["nt"], c["k"])
        mm16.route_groups(s["logits"], ids, wts, score=c["score"], bias=s["bias"], n_group=c["n_group"], top_group=c["top_group"],
                          group_best=c["best"], renorm=c["renorm"], scale=c["scale"])
        return {"ids": ids, "wts": wts}
    if c["op"] == "route_bwd":
        dl = new(c["nt"], c["E"], dtype=torch.float32 if c["d32"] else torch.bfloat16)
        mm16.route_groups_bwd(s["logits"], s["ids"], s["dwts"], dl, score=c["score"], renorm=c["renorm"], scale=c["scale"])
        return {"dlogits": dl}
    if "lora" not in s:
        s["lora"] = mm16.Lora16(s["A"], s["B"], s["scale"])
    out = torch.empty_like(s["base"])
    ws = new(mm16.lora_ws_bytes(s["lora"], c["m"]), dtype=torch.uint8)
    mm16.lora(s["lora"], s["x"], s["ids"], out, resid=s["base"], ws=ws)
    return {"out": out}


# ------------------------------------------------------------------ the plain form

def _scores(c, s):
    """64-bit scores: the order of two experts may hang on their last bits"""
    l = s["logits"].double()
    if c["score"] == "sigmoid":
        return 1 / (1 + torch.exp(-l))
    e = torch.exp(l - l.amax(1, keepdim=True))
    return e / e.sum(1, keepdim=True)


def _best(v, k):
    """indices of the k largest of each row, the lower index first among equals"""
    return torch.sort(v, dim=1, descending=True, stable=True).indices[:, :k]


def _choose(c, s):
    nt, E, G = c["nt"], c["E"], c["n_group"]
    score = _scores(c, s)
    pick = score if s["bias"] is None else score + s["bias"].double()
    if c["top_group"] < G:
        by_group = pick.view(nt, G, E // G)
        worth = torch.sort(by_group, dim=2, descending=True).values[:, :, :c["best"]].sum(2)
        keep = torch.zeros(nt, G, dtype=torch.bool, device=DEV).scatter_(1, _best(worth, c["top_group"]), True)
        pick = torch.where(keep.repeat_interleave(E // G, 1), pick, torch.full_like(pick, -math.inf))
    ids = _best(pick, c["k"])
    return ids, score


def run(state):
    s = state
    if own:
        return _run_own(s)
    c = s["c"]
    if c["op"] == "norm":
        T = TYPES[c["type"]]
        total = None
        x = s["x"]
        if c["add"]:
            total = x = (x.float() + s["add"].float()).to(x.dtype)
        x = x.float()
        mean = x.mean(1, keepdim=True) if c["kind"] == "layer" else 0.0
        xc = x - mean
        rstd = 1 / torch.sqrt((xc * xc).mean(1, keepdim=True) + 1e-5)
        y = xc * rstd * s["w"]
        if s["b"] is not None:
            y = y + s["b"]
        return {"y": y.to(T), "total": total, "mean": mean[:, 0] if c["kind"] == "layer" else None, "rstd": rstd[:, 0]}
    if c["op"] == "norm_bwd":
        x, dy = s["x"].float(), s["dy"].float()
        rstd = s["rstd"][:, None]
        xh = (x - s["mean"][:, None]) * rstd if c["kind"] == "layer" else x * rstd
        g = dy * s["w"]
        dx = g - xh * (g * xh).mean(1, keepdim=True)
        if c["kind"] == "layer":
            dx = dx - g.mean(1, keepdim=True)
        dx = dx * rstd
        if s["resid"] is not None:
            dx = dx + s["resid"].float()
        return {"dx": dx.to(s["x"].dtype), "dw": (dy * xh).sum(0), "db": dy.sum(0) if c["kind"] == "layer" else None}
    if c["op"] == "route":
        ids, score = _choose(c, s)
        w = score.gather(1, ids)
        if c["renorm"]:
            w = w / w.sum(1, keepdim=True)
        return {"ids": ids.to(torch.int32), "wts": (w * c["scale"]).float()}
    if c["op"] == "route_bwd":
        ids, dw = s["ids"].long(), s["dwts"].double()
        score = _scores(c, s)
        chosen = score.gather(1, ids)
        dchosen = dw * c["scale"]
        if c["renorm"]:   # w = scale s / S
            S = chosen.sum(1, keepdim=True)
            dchosen = (dchosen - (dchosen * chosen).sum(1, keepdim=True) / S) / S
        ds = torch.zeros_like(score).scatter_(1, ids, dchosen)
        if c["score"] == "sigmoid":
            dl = ds * score * (1 - score)
        else:
            dl = score * (ds - (ds * score).sum(1, keepdim=True))
        return {"dlogits": dl.to(torch.float32 if c["d32"] else torch.bfloat16)}
    out = s["base"].float()
    if c["lengths"] == "one":   # each row with its own copy of its adapter
        a = s["ids"].clamp_min(0).long()
        low = torch.bmm(s["A"][a].float(), s["x"].float()[:, :, None])
        delta = torch.bmm(s["B"][a].float(), low)[:, :, 0] * s["scale"][a][:, None]
        return {"out": torch.where(s["ids"][:, None] >= 0, out + delta, out).to(s["base"].dtype)}
    for a, first, end in s["prompts"]:
        if a >= 0:
            out[first:end] += s["x"][first:end].float() @ s["A"][a].float().t() @ s["B"][a].float().t() * s["scale"][a]
    return {"out": out.to(s["base"].dtype)}


# ------------------------------------------------------------------ what a pass cannot do without

def work(case):
    c = case
    if c["op"] in ("norm", "norm_bwd"):
        m, n, X = c["m"], c["n"], 4 if c["x32"] else 2
        layer = c["kind"] == "layer"
        if c["op"] == "norm":
            return {"bytes": m * n * (X * (3 if c["add"] else 1) + 2.0) + 4 * n * (2 if layer else 1) + 4 * m * (2 if layer else 1), "flops": 8.0 * m * n}
        return {"bytes": m * n * (X * (3 if c["add"] else 2) + 2.0) + 4 * n * (3 if layer else 2) + 4 * m * (2 if layer else 1), "flops": 14.0 * m * n}
    if c["op"] in ("route", "route_bwd"):
        nt, E, k = c["nt"], c["E"], c["k"]
        if c["op"] == "route":
            return {"bytes": 4.0 * nt * E + 8 * nt * k + (4 * E if c["bias"] else 0), "flops": 20.0 * nt * E}
        # the logits are needed where the sum runs over all of them, else those of the chosen only
        read = E if c["score"] == "softmax" and not c["renorm"] else k
        return {"bytes": 4.0 * nt * read + 8 * nt * k + nt * E * (4 if c["d32"] else 2), "flops": 8.0 * nt * E}
    m, k, n, r = c["m"], c["k"], c["n"], c["r"]
    touched = c["adapters"] * (1 - (1 - 0.875 / c["adapters"]) ** c["requests"])   # expected
    return {"bytes": 2.0 * m * k + m * n * (8.0 if c["f32"] else 4.0) + touched * 2 * r * (k + n) + 4 * m, "flops": 0.875 * 2.0 * m * r * (k + n)}


# ------------------------------------------------------------------ the same in 64 bits

def _exact_route(c, s):
    """scores, then one expert after the other: the best that is left, the lowest index among equals"""
    l = s["logits"].double()
    if c["score"] == "softmax":
        sc = torch.exp(l - torch.logsumexp(l, 1, keepdim=True))
    else:
        sc = torch.where(l >= 0, 1 / (1 + torch.exp(-l.abs())), torch.exp(-l.abs()) / (1 + torch.exp(-l.abs())))
    nt, E, G = c["nt"], c["E"], c["n_group"]
    left = sc + s["bias"].double() if c["bias"] else sc.clone()
    none = torch.full((), -math.inf, dtype=torch.float64, device=DEV)
    at = torch.arange(nt, device=DEV)
    index = torch.arange(E, device=DEV)

    def first_best(v):
        top = v.amax(1, keepdim=True)
        return torch.where(v == top, index[:v.shape[1]], torch.full_like(index[:v.shape[1]], E)).amin(1)
    if c["top_group"] < G:
        grouped = left.view(nt * G, E // G).clone()
        worth = grouped.amax(1)
        if c["best"] == 2:
            rest = grouped
            rest[torch.arange(nt * G, device=DEV), first_best(rest)] = none
            worth = worth + rest.amax(1)
        worth = worth.view(nt, G).clone()
        kept = torch.zeros(nt, G, dtype=torch.bool, device=DEV)
        for _ in range(c["top_group"]):
            i = first_best(worth)
            kept[at, i] = True
            worth[at, i] = none
        left = torch.where(kept[:, index // (E // G)], left, none)
    ids = []
    for _ in range(c["k"]):
        i = first_best(left)
        ids.append(i)
        left[at, i] = none
    return torch.stack(ids, 1), sc


def exact(case, seed):
    c, s = case, prepare(case, seed)
    D = lambda t: t.double()  # noqa: E731
    if c["op"] == "norm":
        x, total = D(s["x"]), None
        if c["add"]:
            total = x + D(s["add"])
            x = D(total.to(s["x"].dtype))   # the rows as they stand in the stream
        mean = x.sum(1) / c["n"] if c["kind"] == "layer" else torch.zeros_like(x[:, 0])
        x = x - mean[:, None]
        rstd = (torch.linalg.vector_norm(x, dim=1) ** 2 / c["n"] + 1e-5) ** -0.5
        y = torch.einsum("ij,i,j->ij", x, rstd, D(s["w"]))
        y = y + D(s["b"]) if c["kind"] == "layer" else y
        return {"y": y, "total": total, "mean": mean if c["kind"] == "layer" else None, "rstd": rstd}
    if c["op"] == "norm_bwd":
        layer = c["kind"] == "layer"
        x, r, n = D(s["x"]), D(s["rstd"])[:, None], c["n"]
        x = x - D(s["mean"])[:, None] if layer else x
        dy, g = D(s["dy"]), D(s["dy"]) * D(s["w"])
        dx = r * g - r ** 3 / n * x * (g * x).sum(1, keepdim=True)
        dx = dx - r / n * g.sum(1, keepdim=True) if layer else dx
        dx = dx + D(s["resid"]) if c["add"] else dx
        return {"dx": dx, "dw": (dy * x * r).sum(0), "db": dy.sum(0) if layer else None}
    if c["op"] == "route":
        ids, sc = _exact_route(c, s)
        w = torch.stack([sc[torch.arange(c["nt"], device=DEV), i] for i in ids.unbind(1)], 1) * c["scale"]
        return {"ids": ids.to(torch.int32), "wts": w / (w.sum(1, keepdim=True) / c["scale"]) if c["renorm"] else w}
    if c["op"] == "route_bwd":
        l, dw = D(s["logits"]), D(s["dwts"])
        at, ids = torch.arange(c["nt"], device=DEV), s["ids"].long()
        out = torch.zeros_like(l)
        z = l.gather(1, ids)
        if c["score"] == "sigmoid":
            sig = 1 / (1 + torch.exp(-z))
            if c["renorm"]:
                w = sig / sig.sum(1, keepdim=True)
                dz = c["scale"] * (1 - sig) * w * (dw - (w * dw).sum(1, keepdim=True))
            else:
                dz = c["scale"] * dw * sig / (1 + torch.exp(z))
        elif c["renorm"]:   # a softmax of the chosen logits
            w = torch.exp(z - torch.logsumexp(z, 1, keepdim=True))
            dz = c["scale"] * w * (dw - (w * dw).sum(1, keepdim=True))
        else:
            p = torch.exp(l - torch.logsumexp(l, 1, keepdim=True))
            pz = p.gather(1, ids)
            out = -c["scale"] * p * (pz * dw).sum(1, keepdim=True)
            dz = c["scale"] * pz * dw
        for j in range(c["k"]):
            out[at, ids[:, j]] += dz[:, j]
        return {"dlogits": out}
    # per row: the base and the row's adapter's product, each adapter's matrices multiplied out for a slice of its rows
    out = D(s["base"])
    for a in s["ids"].unique().tolist():
        if a >= 0:
            rows = (s["ids"] == a).nonzero()[:, 0]
            low = torch.mm(D(s["A"][a]), D(s["x"][rows]).t())
            out[rows] += torch.mm(D(s["B"][a]) * D(s["scale"][a]), low).t()
    return {"out": out}
