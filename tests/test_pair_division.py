"""The kernels' division of a pair by the pairs a token (hyper_amd/csrc/hy_div.h), compiled for the CPU."""
import ctypes
import random
import shutil
import subprocess
from pathlib import Path

import pytest

CSRC = Path(__file__).resolve().parents[1] / "hyper_amd" / "csrc"
SOURCE = """
#define __host__
#define __device__
#include "hy_div.h"
extern "C" int quotient(int p, unsigned k) { return hy::div_k(p, hy::divisor(k)); }
// the first p of a run that goes wrong, -1: none
extern "C" int wrong(int from, int to, unsigned k) {
    const hy::Divisor d = hy::divisor(k);
    for (int p = from; p < to; ++p) if (hy::div_k(p, d) != p / (int) k) return p;
    return -1;
}
"""


@pytest.fixture(scope="module")
def div(tmp_path_factory):
    if not shutil.which("g++"):
        pytest.skip("g++ missing")
    at = tmp_path_factory.mktemp("div")
    (at / "div.cpp").write_text(SOURCE)
    subprocess.run(["g++", "-O2", "-std=c++17", "-shared", "-fPIC", f"-I{CSRC}", str(at / "div.cpp"), "-o", str(at / "div.so")], check=True)
    return ctypes.CDLL(str(at / "div.so"))


def test_quotients(div):
    """every divisor: around the multiples that lie next to a power of two, at the ends of the range, and scattered"""
    rng = random.Random(1)
    for k in range(1, 65):
        at = {0, 1, 2 ** 30 - 1, 2 ** 30, 2 ** 31 - 1, 2 ** 24 * k - 1, 2 ** 24 * k, 2 ** 24 * k + 1} | {rng.randrange(2 ** 31) for _ in range(2000)}
        for e in range(31):
            q = 2 ** e // k * k
            at |= {q - 1, q, q + 1, q + k - 1, q + k}
        for p in sorted(v for v in at if 0 <= v < 2 ** 31):
            assert div.quotient(p, k) == p // k, (p, k)


@pytest.mark.parametrize("k", [1, 2, 3, 7, 8, 10, 33, 63, 64])
def test_runs(div, k):
    for start in (0, 2 ** 24 * k - 50000, 2 ** 30, 2 ** 31 - 100001):
        start = min(start, 2 ** 31 - 100001)
        assert div.wrong(start, start + 100000, k) == -1
