"""The waits that matrix instructions need around them, in the built code.  The 256 x 256 tiles issue theirs as inline assembly,
where the compiler adds no waits: their operands come from LDS reads and their sums are read behind explicit waits, and what
lies between is up to the compiler's schedule.  Read from the disassembly of libhymoe.so's 16-bit products:

  a vector instruction's result is an operand no sooner than 2 wait states behind it (4 behind one that writes the lane mask);
  a product of 16 x 16 x 32 (8 passes) is read by anything but a product no sooner than 11 wait states behind it.

An instruction is one wait state, s_nop N is N + 1.  Paths: straight on, and over each branch to its target."""
import re
import shutil
import struct
import subprocess
from pathlib import Path

import pytest

import hyper_amd.build

OBJDUMP = shutil.which("llvm-objdump") or "/opt/rocm/llvm/bin/llvm-objdump"
REG = re.compile(r"^\|?-?([va])(?:(\d+)|\[(\d+):(\d+)\])\|?$")
OPERAND, MASK, RESULT = 2, 4, 11


def regs(token):
    m = REG.match(token.strip())
    if not m:
        return frozenset()
    lo, hi = (int(m[2]), int(m[2])) if m[2] else (int(m[3]), int(m[4]))
    return frozenset((m[1], i) for i in range(lo, hi + 1))


class Op:
    """one instruction: what it writes and reads of vector registers, the wait states it stands for"""

    def __init__(self, name, args):
        self.name, t = name, [regs(a) for a in args]
        self.mfma, self.valu = name.startswith(("v_mfma", "v_smfmac")), name.startswith("v_")
        store = name.startswith(("ds_write", "global_store", "buffer_store", "flat_store", "scratch_store"))
        self.writes = t[0] if t and not store else frozenset()
        if name.startswith(("v_swap", "v_permlane16_swap", "v_permlane32_swap")):
            self.writes = t[0] | t[1]
        self.reads = frozenset().union(*(t if store else t[1:])) if t else frozenset()
        if name.startswith(("v_fmac", "v_swap", "v_permlane", "v_dot2c", "v_dot4c", "v_mov_b32_dpp", "ds_", "global_", "buffer_")):
            self.reads |= self.writes
        self.states = int(args[0], 0) + 1 if name == "s_nop" else 1
        self.mask = name.startswith("v_cmpx")


def faults(before, ops):
    """hazards at ops, whose predecessors on the path are `before`"""
    path, out = list(before), []
    for op in ops:
        d = 0
        for p in reversed(path):
            if d >= RESULT:
                break
            if op.mfma and p.valu and not p.mfma and ((d < OPERAND and p.writes & op.reads) or (d < MASK and p.mask)):
                out.append(f"{p.name} -> {op.name}: {d} wait states")
            if p.mfma and not op.mfma and p.writes & op.reads:
                out.append(f"{p.name} -> {op.name}: {d} wait states")
            d += p.states
        path.append(op)
        path = path[-RESULT:]
    return out


def kernels(text):
    """name -> [(address, Op, branch target)] of a disassembly"""
    out, at = {}, None
    for line in text.splitlines():
        m = re.match(r"^([0-9a-f]+) <(.+)>:$", line)
        if m:
            at = out.setdefault(m[2], [])
            base = int(m[1], 16)
            continue
        m = re.match(r"^\s+(\S+)\s*(.*?)\s*// ([0-9A-F]+):", line)
        if not m or at is None:
            continue
        to = re.search(r"<[^>]+\+0x([0-9a-f]+)>$", line) if m[1].startswith(("s_cbranch", "s_branch")) else None
        at.append((int(m[3], 16), Op(m[1], [a for a in m[2].split(",") if a]), base + int(to[1], 16) if to else None))
    return out


def check(code):
    """the number of products and the hazards of a kernel"""
    ops, index = [c[1] for c in code], {c[0]: i for i, c in enumerate(code)}
    bad = faults([], ops)
    for i, (_, _, to) in enumerate(code):
        if to is not None and to in index:
            j = index[to]
            bad += faults(ops[max(0, i + 1 - RESULT):i + 1], ops[j:j + RESULT])
    return sum(o.mfma for o in ops), bad


def code_objects(lib):
    at = 0
    while (at := lib.find(b"__CLANG_OFFLOAD_BUNDLE__", at)) >= 0:
        n, = struct.unpack_from("<Q", lib, at + 24)
        p = at + 32
        for _ in range(n):
            off, size, tl = struct.unpack_from("<QQQ", lib, p)
            if b"amdgcn" in lib[p + 24:p + 24 + tl] and size:
                yield lib[at + off:at + off + size]
            p += 24 + tl
        at += 24


def test_the_rules_find_what_breaks_them():
    """on written-out code: each rule, each path"""
    def code(*lines):
        out = []
        for i, (text, to) in enumerate(lines):
            name, _, rest = text.partition(" ")
            out.append((4 * i, Op(name, rest.split(",") if rest else []), to))
        return out
    product = ("v_mfma_f32_16x16x32_bf16 a[0:3], v[0:3], v[4:7], a[0:3]", None)
    move, other, nop = ("v_mov_b32_e32 v5, v9", None), ("v_mov_b32_e32 v20, v9", None), ("s_nop 0", None)
    assert check(code(move, product))[1] and check(code(move, other, product))[1] and not check(code(move, other, nop, product))[1]
    assert check(code(("v_accvgpr_write_b32 a2, 0", None), nop, product))[1]
    assert check(code(("v_cmpx_lt_i32_e32 v20, v21", None), nop, nop, product))[1]
    assert not check(code(("ds_read_b128 v[0:3], v9", None), product))[1]
    read, store = ("v_accvgpr_read_b32 v30, a1", None), ("ds_write_b128 v30, a[0:3]", None)
    wait = ("s_nop 9", None)
    for use in (read, store):
        assert check(code(product, wait, use))[1] and not check(code(product, ("s_nop 10", None), use))[1]
    assert not check(code(product, product))[1]
    assert check(code(product, nop, nop, nop, nop, nop, move, ("s_cbranch_scc1 0", 0)))[1]          # over the loop's end
    assert not check(code(product, nop, nop, nop, nop, nop, move, nop, ("s_cbranch_scc1 0", 0)))[1]


def test_products_of_the_built_library():
    if not Path(OBJDUMP).exists():
        pytest.skip("llvm-objdump missing")
    found, asm = 0, 0
    for obj in code_objects(hyper_amd.build.OUT.read_bytes()):
        if b"k_mm" not in obj and b"k_few" not in obj:
            continue
        r = subprocess.run([OBJDUMP, "-d", "--mcpu=gfx950", "-"], input=obj, capture_output=True)
        assert r.returncode == 0, r.stderr
        for name, code in kernels(r.stdout.decode()).items():
            n, bad = check(code)
            found += n
            asm += "k_gradients" in name and n > 0
            assert not bad, (name, bad[:3])
    assert found > 3000 and asm >= 4
