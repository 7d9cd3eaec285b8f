"""16-bit (bf16 / fp16) matrix products on torch device tensors: linear layers with bias, activation and residual, products
grouped by expert, and their gradients -- for experts, shared experts and dense layers that GGUF files hold as F16 or BF16.

The functions call libhymoe's C ABI (include/hymoe.h) and write into tensors the caller owns; a mistake in the arguments
raises ValueError here or HyError from the library.  They run on `stream` (None: the current stream of the tensors'
device).  Matrices are row-major with contiguous rows; rows may lie apart (views of wider tensors).

Moe16LayerRunner strings them together for one layer: router, routing, grouping, gate/up, down, combine, and the backward
pass of the experts.
"""
import ctypes
from typing import Optional

import numpy as np
import torch

from . import check, hy_moe_dev, lib
from . import moe

HY_F32, HY_F16, HY_BF16 = 0, 1, 30
_TYPE = {torch.float32: HY_F32, torch.float16: HY_F16, torch.bfloat16: HY_BF16}
ACTS = {"none": 0, "relu": 1, "silu": 2, "gelu": 3, "gelu_tanh": 4}


def _type16(t: torch.Tensor) -> int:
    v = _TYPE.get(t.dtype)
    if v != HY_BF16 and v != HY_F16:
        raise ValueError(f"expected bfloat16 or float16, got {t.dtype}")
    return v


def _p(t: Optional[torch.Tensor]):
    return None if t is None else t.data_ptr()


def _call(fn, ref: torch.Tensor, stream, others, *args) -> None:
    """fn(*args, stream) on ref's GPU, which is current while the call launches; every tensor must be on it.  (Written for
    few Python steps: a decode call's kernel takes about as long as its checks.)"""
    dev = ref.get_device()
    if dev < 0:
        raise ValueError(f"tensors must be on a GPU, got {ref.device}")
    for t in others:
        if t is not None and t.get_device() != dev:
            raise ValueError(f"tensors on {ref.device} and {t.device}")
    if stream is None:
        raw = torch._C._cuda_getCurrentRawStream(dev)
    elif stream.device_index != dev:
        raise ValueError(f"a stream of cuda:{stream.device_index} for tensors on {ref.device}")
    else:
        raw = stream.cuda_stream
    if dev == torch._C._cuda_getDevice():
        rc = fn(*args, raw)
    else:
        with torch.cuda.device(dev):
            rc = fn(*args, raw)
    if rc:
        check(rc)


def _mat(name: str, t: torch.Tensor, rows: Optional[int], cols: int, *dtypes, least: bool = False) -> int:
    """checks a row-major matrix and returns the elements between its rows (least: it may have more rows)"""
    shape = t.shape
    if shape == (rows, cols) and (not dtypes or t.dtype in dtypes):   # the usual case
        between, step = t.stride()
        if step == 1:
            return between if rows > 1 else cols
    if len(shape) != 2 or shape[1] != cols or (rows is not None and (shape[0] < rows if least else shape[0] != rows)):
        raise ValueError(f"{name} must be [{'*' if rows is None else rows}, {cols}], got {tuple(shape)}")
    if dtypes and t.dtype not in dtypes:
        raise ValueError(f"{name} must be {' or '.join(str(d) for d in dtypes)}, got {t.dtype}")
    between, step = t.stride()
    if step != 1 and cols > 1:
        raise ValueError(f"{name} must have contiguous rows")
    return between if shape[0] > 1 else cols


def _vec(name: str, t: Optional[torch.Tensor], n: int, dtype) -> None:
    if t is not None and (t.dtype != dtype or t.numel() < n or not t.is_contiguous()):
        raise ValueError(f"{name} must hold {n} contiguous {dtype} values, got {t.dtype} {tuple(t.shape)}")


def _act(act: str) -> int:
    v = ACTS.get(act)
    if v is None:
        raise ValueError(f"unknown activation {act!r}")
    return v


# ------------------------------------------------------------------ linear layers

def linear(W, x, out, bias=None, act="none", resid=None, z=None, stream=None):
    """out = act(x W^T + bias) + resid for x [m, k], W [n, k]; out (and resid) of the operands' type or float32, bias
    float32, z the pre-activation kept for act_bwd.  resid may be out itself."""
    dt, (n, k), m = W.dtype, W.shape, x.shape[0]
    ldw, ldx = _mat("W", W, n, k), _mat("x", x, m, k, dt)
    ldo = _mat("out", out, m, n, dt, torch.float32)
    ldr = _mat("resid", resid, m, n, out.dtype) if resid is not None else 0
    ldz = _mat("z", z, m, n, dt) if z is not None else 0
    if bias is not None:
        _vec("bias", bias, n, torch.float32)
    _call(lib().hy_linear, W, stream, (x, out, bias, resid, z),
          _type16(W), W.data_ptr(), ldw, n, k, x.data_ptr(), ldx, m, _p(bias), _act(act), _p(resid), ldr, _p(z), ldz, out.data_ptr(),
          _TYPE[out.dtype], ldo)


def linear_glu(Wg, Wu, x, h, clamp=0.0, g=None, u=None, stream=None):
    """h = silu(x Wg^T) (x Wu^T), with the SwiGLU limit `clamp` (0: none); g and u keep the two products for swiglu_bwd."""
    ty, (n, k), m = _type16(Wg), Wg.shape, x.shape[0]
    ldw = _mat("Wg", Wg, n, k)
    if _mat("Wu", Wu, n, k, Wg.dtype) != ldw:
        raise ValueError("Wg and Wu must have the same row stride")
    ldx, ldh = _mat("x", x, m, k, Wg.dtype), _mat("h", h, m, n, Wg.dtype)
    for name, t in (("g", g), ("u", u)):
        if t is not None and _mat(name, t, m, n, Wg.dtype) != ldh:
            raise ValueError(f"{name} must have h's row stride")
    _call(lib().hy_linear_glu, Wg, stream, (Wu, x, h, g, u),
          ty, _p(Wg), _p(Wu), ldw, n, k, _p(x), ldx, m, float(clamp), _p(g), _p(u), _p(h), ldh)


def act_bwd(act, z, dy, dz, stream=None):
    """dz = dy act'(z), all [m, n] of one 16-bit type."""
    ty, (m, n) = _type16(z), z.shape
    ldz, ldd, ldo = _mat("z", z, m, n), _mat("dy", dy, m, n, z.dtype), _mat("dz", dz, m, n, z.dtype)
    _call(lib().hy_act_bwd, z, stream, (dy, dz), ty, _act(act), _p(z), ldz, _p(dy), ldd, m, n, _p(dz), ldo)


def linear_dx(W, dz, dx, resid=None, stream=None):
    """dx = dz W + resid for dz [m, n], W [n, k]."""
    ty, (n, k), m = _type16(W), W.shape, dz.shape[0]
    ldw, ldd = _mat("W", W, n, k), _mat("dz", dz, m, n, W.dtype)
    ldo = _mat("dx", dx, m, k, W.dtype, torch.float32)
    ldr = _mat("resid", resid, m, k, dx.dtype) if resid is not None else 0
    _call(lib().hy_linear_dx, W, stream, (dz, dx, resid),
          ty, _p(W), ldw, n, k, _p(dz), ldd, m, _p(resid), ldr, _p(dx), _TYPE[dx.dtype], ldo)


def linear_dw_ws_bytes(m: int, n: int, k: int) -> int:
    """bytes of linear_dw's workspace (0: none needed)"""
    return lib().hy_linear_dw_ws_bytes(m, n, k)


def linear_dw(dz, x, dW, db=None, accumulate=False, ws=None, stream=None):
    """dW = dz^T x [n, k] and db = the column sums of dz (float32), added to what is there with `accumulate`.  ws: a uint8
    tensor of linear_dw_ws_bytes(m, n, k) bytes, free again once the call's work on the stream is done."""
    ty, (m, n), k = _type16(dz), dz.shape, x.shape[-1]
    ldd, ldx = _mat("dz", dz, m, n), _mat("x", x, m, k, dz.dtype)
    ldw = _mat("dW", dW, n, k, dz.dtype, torch.float32)
    _vec("db", db, n, torch.float32)
    _vec("ws", ws, 0, torch.uint8)
    _call(lib().hy_linear_dw, dW, stream, (dz, x, db, ws),
          ty, _p(dz), ldd, _p(x), ldx, m, n, k, _p(dW), _TYPE[dW.dtype], ldw, _p(db), int(bool(accumulate)), _p(ws),
          0 if ws is None else ws.numel())


def rows16(x, out, stream=None):
    """float32 rows rounded to out's 16-bit type."""
    ty, (m, n) = _type16(out), out.shape
    xs, ldo = _mat("x", x, m, n, torch.float32), _mat("out", out, m, n)
    _call(lib().hy_rows16, out, stream, (x,), ty, _p(x), xs, n, m, _p(out), ldo)


# ------------------------------------------------------------------ experts

class Moe16Dev:
    """Experts of one layer in 16 bits: gate, up [E, ff, n] and down [E, n, ff], contiguous, and the slot table (int32, one
    entry an expert: its local matrix or -1).  Keeps the tensors alive; moe.moe_order takes it as it takes a MoeDev.
    gate/up or down may be None for calls that do not read them."""

    def __init__(self, gate, up, down, slot: torch.Tensor, clamp: float = 0.0):
        c = hy_moe_dev()
        shape = None
        for name, t, flip in (("gate", gate, False), ("up", up, False), ("down", down, True)):
            if t is None:
                continue
            if t.dim() != 3 or not t.is_contiguous():
                raise ValueError(f"{name} must be a contiguous [E, rows, cols] tensor")
            E, a, b = t.shape
            s = (E, b, a) if flip else (E, a, b)
            if shape not in (None, s):
                raise ValueError(f"{name} {tuple(t.shape)} does not fit the other matrices")
            shape = s
            setattr(c, name, t.data_ptr())
        if shape is None or (gate is None) != (up is None):
            raise ValueError("gate and up, down, or all three are needed")
        if gate is not None and gate.dtype != up.dtype:
            raise ValueError("gate and up must have one type")
        _vec("slot", slot, 1, torch.int32)
        for t in (gate, up, down):
            if t is not None and t.device != slot.device:
                raise ValueError(f"matrices on {t.device}, slot on {slot.device}")
        self.gate, self.up, self.down, self.slot, self.clamp = gate, up, down, slot, float(clamp)
        c.n_local, c.ff, c.n = shape
        self.n_local, self.ff, self.n = shape
        c.tg = _type16(gate) if gate is not None else _type16(down)
        c.td = _type16(down) if down is not None else c.tg
        c.gate_bytes = c.down_bytes = 2 * self.ff * self.n
        c.slot, c.n_expert, c.clamp = slot.data_ptr(), slot.numel(), self.clamp
        self.c = c
        self.ref = ctypes.byref(c)


def experts_from_gguf(g, il: int, device="cuda", clamp: float = 0.0) -> Moe16Dev:
    """Layer il's routed experts (blk.<il>.ffn_{gate,up,down}_exps.weight, F16 or BF16) on the device, every expert local."""
    mats = []
    for part in ("gate", "up", "down"):
        t = g.need(f"blk.{il}.ffn_{part}_exps.weight")
        dt = {HY_F16: torch.float16, HY_BF16: torch.bfloat16}.get(int(t.type))
        if dt is None:
            raise ValueError(f"{t.name}: type {int(t.type)} is not F16 or BF16")
        ne = list(t.ne) + [1] * (3 - len(t.ne))
        raw = torch.from_numpy(np.array(t.data()))   # a copy of the mapped bytes
        mats.append(raw.view(dt).reshape(ne[2], ne[1], ne[0]).to(device))
    return Moe16Dev(*mats, torch.arange(mats[0].shape[0], dtype=torch.int32, device=device), clamp)


def _groups(n_pairs, ids, order, order_n, egrp, max_active):
    if order is None:
        if ids is not None:
            _vec("ids", ids, n_pairs, torch.int32)
        return
    _vec("order", order, n_pairs, torch.int32)
    _vec("order_n", order_n, 2 if n_pairs else 0, torch.int32)   # (no pairs: nothing reads them)
    _vec("egrp", egrp, 3 * max_active if n_pairs else 0, torch.int32)


def _pairs(name, t, rows, cols, *dtypes):
    if t.shape == (rows, cols) and t.dtype in dtypes and t.is_contiguous():   # the usual case
        return
    if _mat(name, t, rows, cols, *dtypes, least=True) != cols:
        raise ValueError(f"{name} must be contiguous")


def moe16_gate_up(m: Moe16Dev, x, k, n_pairs, h, ids=None, order=None, order_n=None, egrp=None, max_active=0, g=None, u=None, stream=None):
    """h[p] = SwiGLU(gate_e x[p // k], up_e x[p // k]); g and u keep the products.  Grouped (order, order_n, egrp of
    moe.moe_order) or, without order, each pair by its expert ids[p]."""
    if m.gate is None:
        raise ValueError("the experts have no gate/up")
    dt = m.gate.dtype
    ldx = _mat("x", x, (n_pairs + k - 1) // max(k, 1), m.n, dt, least=True)
    for name, t in (("h", h), ("g", g), ("u", u)):
        if t is not None:
            _pairs(name, t, n_pairs, m.ff, dt)
    _groups(n_pairs, ids, order, order_n, egrp, max_active)
    _call(lib().hy_moe16_gate_up, m.slot, stream, (x, h, ids, order, order_n, egrp, g, u),
          m.ref, _p(x), ldx, k, _p(ids), n_pairs, _p(order), _p(order_n), _p(egrp), max_active, _p(g), _p(u), _p(h))


def moe16_down(m: Moe16Dev, h, n_pairs, y, wts=None, ids=None, order=None, order_n=None, egrp=None, max_active=0, stream=None):
    """y[p] = wts[p] (down_e h[p]), y of the experts' type or float32."""
    if m.down is None:
        raise ValueError("the experts have no down")
    dt = m.down.dtype
    _pairs("h", h, n_pairs, m.ff, dt)
    _pairs("y", y, n_pairs, m.n, dt, torch.float32)
    _vec("wts", wts, n_pairs, torch.float32)
    _groups(n_pairs, ids, order, order_n, egrp, max_active)
    _call(lib().hy_moe16_down, m.slot, stream, (h, y, wts, ids, order, order_n, egrp),
          m.ref, _p(h), _p(ids), n_pairs, _p(order), _p(order_n), _p(egrp), max_active, _p(wts), _p(y), _TYPE[y.dtype])


def moe16_reduce(m: Moe16Dev, shexp, sg, y, k, out, nt, ids, stream=None):
    """out[t] = sg[t] shexp[t] + the float32 rows y of token t's pairs, in ascending expert order, pairs whose expert is not
    local left out; shexp and sg may be None."""
    _pairs("y", y, nt * k, m.n, torch.float32)
    _pairs("out", out, nt, m.n, torch.float32)
    if shexp is not None:
        _pairs("shexp", shexp, nt, m.n, torch.float32)
    _vec("sg", sg, nt, torch.float32)
    _vec("ids", ids, nt * k, torch.int32)
    _call(lib().hy_moe16_reduce, m.slot, stream, (shexp, sg, y, out, ids), m.ref, _p(shexp), _p(sg), _p(y), k, _p(out), nt, _p(ids))


def moe16_down_dx(m: Moe16Dev, dy, k, n_pairs, order, order_n, egrp, max_active, dh, stream=None):
    """dh[p] = dy[p // k] down_e, not yet weighted."""
    if m.down is None:
        raise ValueError("the experts have no down")
    dt = m.down.dtype
    ldd = _mat("dy", dy, (n_pairs + k - 1) // max(k, 1), m.n, dt, least=True)
    _pairs("dh", dh, n_pairs, m.ff, dt, torch.float32)
    _groups(n_pairs, None, order, order_n, egrp, max_active)
    _call(lib().hy_moe16_down_dx, m.slot, stream, (dy, dh, order, order_n, egrp),
          m.ref, _p(dy), ldd, k, n_pairs, _p(order), _p(order_n), _p(egrp), max_active, _p(dh), _TYPE[dh.dtype])


def moe16_gate_up_dx(m: Moe16Dev, dg, du, n_pairs, order, order_n, egrp, max_active, dx, stream=None):
    """dx[p] = dg[p] gate_e + du[p] up_e (moe.moe_reduce sums the pairs of a token)."""
    if m.gate is None:
        raise ValueError("the experts have no gate/up")
    dt = m.gate.dtype
    _pairs("dg", dg, n_pairs, m.ff, dt)
    _pairs("du", du, n_pairs, m.ff, dt)
    _pairs("dx", dx, n_pairs, m.n, dt, torch.float32)
    _groups(n_pairs, None, order, order_n, egrp, max_active)
    _call(lib().hy_moe16_gate_up_dx, m.slot, stream, (dg, du, dx, order, order_n, egrp),
          m.ref, _p(dg), _p(du), n_pairs, _p(order), _p(order_n), _p(egrp), max_active, _p(dx), _TYPE[dx.dtype])


def moe16_dw(m: Moe16Dev, a, ka, b, kb, n_pairs, order, order_n, egrp, max_active, dW, accumulate=False, stream=None):
    """dW[slot[e]] = sum over e's pairs of a[p // ka]^T b[p // kb], [n_local, rows, cols]; zeros for a matrix without pairs,
    the sum of them all where experts share one."""
    ty, rows, cols = _type16(a), a.shape[-1], b.shape[-1]
    lda = _mat("a", a, (n_pairs + ka - 1) // max(ka, 1), rows, least=True)
    ldb = _mat("b", b, (n_pairs + kb - 1) // max(kb, 1), cols, a.dtype, least=True)
    if tuple(dW.shape) != (m.n_local, rows, cols) or not dW.is_contiguous() or dW.dtype not in (a.dtype, torch.float32):
        raise ValueError(f"dW must be contiguous [{m.n_local}, {rows}, {cols}] of {a.dtype} or float32, got {dW.dtype} {tuple(dW.shape)}")
    _groups(n_pairs, None, order, order_n, egrp, max_active)
    _call(lib().hy_moe16_dw, m.slot, stream, (a, b, dW, order, order_n, egrp),
          m.ref, ty, _p(a), lda, ka, rows, _p(b), ldb, kb, cols, n_pairs, _p(order), _p(order_n), _p(egrp), max_active, _p(dW),
          _TYPE[dW.dtype], int(bool(accumulate)))


def swiglu_bwd(g, u, dh, wts, dg, du, hw=None, dwts=None, clamp=0.0, order=None, order_n=None, stream=None):
    """From g, u [P, ff] and the unweighted dh: dg, du, hw = wts h and dwts[p] = sum dh h (the pairs of order, or all)."""
    shape, dt = g.shape, g.dtype
    for t in (g, u, dh, dg, du, hw):
        if t is not None and not (t.shape == shape and t.dtype is dt and t.is_contiguous()):
            raise ValueError(f"g, u, dh, dg, du and hw must be contiguous matrices of one shape and type, got {t.dtype} {tuple(t.shape)} beside "
                             f"{dt} {tuple(shape)}")
    if len(shape) != 2:
        raise ValueError(f"g must be [pairs, ff], got {tuple(shape)}")
    P, ff = shape
    _vec("wts", wts, P, torch.float32)
    _vec("dwts", dwts, P, torch.float32)
    if order is not None or order_n is not None:
        _vec("order", order, P, torch.int32)
        _vec("order_n", order_n, 1, torch.int32)
    _call(lib().hy_swiglu_bwd, g, stream, (u, dh, wts, dg, du, hw, dwts, order, order_n),
          _type16(g), g.data_ptr(), u.data_ptr(), dh.data_ptr(), _p(wts), P, ff, clamp, _p(order), _p(order_n), dg.data_ptr(), du.data_ptr(),
          _p(hw), _p(dwts))


# ------------------------------------------------------------------ one MoE layer

class Moe16LayerRunner:
    """Workspace and call sequence for one MoE layer with 16-bit experts, as moe.MoeLayerRunner has it for quantized ones:
    router GEMV, softmax routing, then by ids (up to `decode_rows` rows) or grouped: gate/up, down, combine.

    forward(x) takes [nt, d] float32 rows; pairs whose expert dev.slot does not hold at the time add nothing to the output.  With
    keep=True it keeps what backward(dy) needs, the slot table among it; backward is for layers whose experts were all local
    when the runner was made.  `shared`: an always-on expert (a Moe16Dev with one matrix) added with weight 1; backward leaves it
    and the router out."""

    decode_rows = 2   # by ids every pair reads its expert's matrices; grouped, an expert's rows share them

    def __init__(self, dev: Moe16Dev, W_r: torch.Tensor, k: int, max_rows: int, shared: Optional[Moe16Dev] = None):
        if dev.gate is None or dev.down is None or dev.gate.dtype != dev.down.dtype:
            raise ValueError("the experts need gate, up and down of one type")
        if W_r.dtype not in (torch.float32, torch.bfloat16) or W_r.dim() != 2 or not W_r.is_contiguous() or \
                tuple(W_r.shape) != (dev.slot.numel(), dev.n):
            raise ValueError(f"W_r must be a contiguous fp32 or bf16 [{dev.slot.numel()}, {dev.n}] matrix, got {W_r.dtype} {tuple(W_r.shape)}")
        if dev.n % 4:
            raise ValueError("the router takes d_model in multiples of 4")
        if max_rows >= 1 << 23 or -(-dev.slot.numel() // 16) * -(-max_rows // 8) >= 1 << 24:   # (a launch counts its threads in 32 bits)
            raise ValueError(f"max_rows {max_rows} with {dev.slot.numel()} experts: more than the router takes in one launch")
        if shared is not None and (shared.gate is None or shared.down is None or shared.n != dev.n or shared.gate.dtype != dev.gate.dtype
                                   or shared.down.dtype != dev.gate.dtype):
            raise ValueError("the shared expert must have the experts' d_model and type")
        self.dev, self.W_r, self.k, self.shared, self.max_rows = dev, W_r, k, shared, int(max_rows)
        self.E, self.d, self.ff, self.dtype, device = dev.slot.numel(), dev.n, dev.ff, dev.gate.dtype, W_r.device
        T, P = self.max_rows, self.max_rows * k
        new = lambda *s, dtype=self.dtype: torch.empty(*s, dtype=dtype, device=device)  # noqa: E731
        self.logits, self.ids, self.wts = new(T, self.E, dtype=torch.float32), new(P, dtype=torch.int32), new(P, dtype=torch.float32)
        self.order, self.order_n, self.egrp = new(P, dtype=torch.int32), torch.zeros(2, dtype=torch.int32, device=device), new(3 * self.E, dtype=torch.int32)
        self.all_local = bool((dev.slot >= 0).all()) and bool((dev.slot < dev.n_local).all())   # now; every call reads the table itself
        self.x16, self.h, self.y = new(T, self.d), new(P, self.ff), new(P, self.d, dtype=torch.float32)
        self.out = new(T, self.d, dtype=torch.float32)
        self.sh_y = new(T, self.d, dtype=torch.float32) if shared is not None else None
        self.sh_h = new(T, shared.ff) if shared is not None else None
        self.g = self.u = self.kept_dev = None
        self.kept = None   # rows of the last forward(keep=True); None: there was another one since, or none

    def _rows(self, x):
        if x.dim() != 2 or x.shape[1] != self.d or x.dtype != torch.float32 or x.device != self.W_r.device:
            raise ValueError(f"x must be float32 [nt, {self.d}] on {self.W_r.device}")
        if x.shape[0] > self.max_rows:
            raise ValueError(f"{x.shape[0]} rows exceed the runner's max_rows {self.max_rows}")
        if x.stride(1) != 1 or x.stride(0) % 4 or x.data_ptr() % 16:
            raise ValueError("x rows must be contiguous and 16-byte aligned")
        return x.shape[0]

    def _group(self, nt, stream):
        moe.moe_order(self.dev, self.ids, nt * self.k, self.E, self.order, self.order_n, stream, self.egrp)
        return dict(order=self.order, order_n=self.order_n, egrp=self.egrp, max_active=min(self.E, nt * self.k, 1024))

    def forward(self, x: torch.Tensor, keep: bool = False, stream=None) -> torch.Tensor:
        """The layer's output [nt, d] (a view of the runner's buffer) for nt rows; keep=True: also what backward needs."""
        nt, k = self._rows(x), self.k
        P = nt * k
        self.kept = None
        device = self.W_r.device
        stream = stream if stream is not None else torch.cuda.current_stream(device)
        with torch.cuda.stream(stream):
            if keep and self.g is None:
                self.g, self.u = torch.empty_like(self.h), torch.empty_like(self.h)
                self.kept_dev = Moe16Dev(self.dev.gate, self.dev.up, self.dev.down, torch.empty_like(self.dev.slot), self.dev.clamp)
            if nt == 0:
                self.kept = 0 if keep else None
                return self.out[:0]
            moe.gemv_f32(self.W_r, self.E, self.d, x, x.stride(0), self.logits, self.E, nt, stream)
            moe.moe_route(self.logits, self.E, self.E, k, self.ids, self.wts, None, nt, stream)
            rows16(x, self.x16[:nt], stream)
            how = dict(ids=self.ids) if nt <= self.decode_rows and not keep else self._group(nt, stream)
            gu = {}
            if keep:
                gu = dict(g=self.g, u=self.u)
                torch.add(self.dev.slot, 0, out=self.kept_dev.slot)   # (a kernel: no copy node in a captured graph)
            moe16_gate_up(self.dev, self.x16[:nt], k, P, self.h, **how, **gu, stream=stream)
            moe16_down(self.dev, self.h, P, self.y, wts=self.wts, **how, stream=stream)
            if self.shared is not None:
                S = self.shared
                linear_glu(S.gate[0], S.up[0], self.x16[:nt], self.sh_h[:nt], clamp=S.clamp, stream=stream)
                linear(S.down[0], self.sh_h[:nt], self.sh_y[:nt], stream=stream)
            moe16_reduce(self.dev, self.sh_y, None, self.y, k, self.out, nt, self.ids, stream)
        self.kept = nt if keep else None
        return self.out[:nt]

    def backward(self, dy: torch.Tensor, stream=None) -> dict:
        """Gradients of the routed experts for the last forward(keep=True): dy [nt, d] float32 -> {"dx": [nt, d] float32 (the
        experts' part), "dwts": [nt, k] (of the routing weights), "gate", "up", "down": float32}."""
        nt, k = self._rows(dy), self.k
        if nt != self.kept:
            raise ValueError("backward follows forward(keep=True) of the same rows")
        if not self.all_local:
            raise ValueError("backward needs every expert local")
        P, dev = nt * k, self.kept_dev   # the slot table as forward found it
        grp = (self.order, self.order_n, self.egrp, min(self.E, P, 1024))
        new = lambda *s, dtype=self.dtype: torch.empty(*s, dtype=dtype, device=dy.device)  # noqa: E731
        with torch.cuda.stream(stream if stream is not None else torch.cuda.current_stream(dy.device)):
            dy16, dh, dg, du, hw = new(nt, self.d), new(P, self.ff), new(P, self.ff), new(P, self.ff), new(P, self.ff)
            dwts, dxp, dx = torch.zeros(nt, k, device=dy.device), new(P, self.d, dtype=torch.float32), new(nt, self.d, dtype=torch.float32)
            W = {n: new(*t.shape, dtype=torch.float32) for n, t in (("gate", dev.gate), ("up", dev.up), ("down", dev.down))}
            rows16(dy, dy16)
            moe16_down_dx(dev, dy16, k, P, *grp, dh)
            swiglu_bwd(self.g[:P], self.u[:P], dh, self.wts[:P], dg, du, hw, dwts.view(-1), clamp=dev.clamp,
                       order=self.order, order_n=self.order_n)
            moe16_gate_up_dx(dev, dg, du, P, *grp, dxp)
            moe16_reduce(dev, None, None, dxp, k, dx, nt, self.ids)
            moe16_dw(dev, dg, 1, self.x16[:nt], k, P, *grp, W["gate"])
            moe16_dw(dev, du, 1, self.x16[:nt], k, P, *grp, W["up"])
            moe16_dw(dev, dy16, k, hw, 1, P, *grp, W["down"])
        return {"dx": dx, "dwts": dwts, **W}
