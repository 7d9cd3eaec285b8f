"""include/hymoe.hpp's wrappers of the 16-bit products: a program that calls each links against the library, and what the C
entry refuses arrives as an exception with its message."""
import re
import shutil
import subprocess
from pathlib import Path

import pytest

ROOT = Path(__file__).resolve().parents[1]
# a call that is refused for its type or its missing layer, before anything is read
CALLS = {
    "linear": "linear(7, 0, 8, 8, 8, 0, 8, 1, 0, 0, 0, 0, 0, 0, 0, 0, 8, 0)",
    "linear_glu": "linear_glu(7, 0, 0, 8, 8, 8, 0, 8, 1, 0.0f, 0, 0, 0, 8, 0)",
    "act_bwd": "act_bwd(7, 0, 0, 8, 0, 8, 1, 8, 0, 8, 0)",
    "linear_dx": "linear_dx(7, 0, 8, 8, 8, 0, 8, 1, 0, 0, 0, 0, 8, 0)",
    "linear_dw": "linear_dw(7, 0, 8, 0, 8, 1, 8, 8, 0, 0, 8, 0, false, 0, 0, 0)",
    "moe16_gate_up": "moe16_gate_up(m, 0, 8, 2, 0, 4, 0, 0, 0, 1, 0, 0, 0, 0)",
    "moe16_down": "moe16_down(m, 0, 0, 4, 0, 0, 0, 1, 0, 0, 0, 0)",
    "moe16_reduce": "moe16_reduce(m, 0, 0, 0, 2, 0, 1, 0, 0)",
    "moe16_down_dx": "moe16_down_dx(m, 0, 8, 2, 4, 0, 0, 0, 1, 0, 0, 0)",
    "moe16_gate_up_dx": "moe16_gate_up_dx(m, 0, 0, 4, 0, 0, 0, 1, 0, 0, 0)",
    "moe16_dw": "moe16_dw(m, 7, 0, 8, 1, 8, 0, 8, 1, 8, 4, 0, 0, 0, 1, 0, 0, false, 0)",
    "swiglu_bwd": "swiglu_bwd(7, 0, 0, 0, 0, 1, 8, 0.0f, 0, 0, 0, 0, 0, 0, 0)",
    "rows16": "rows16(7, 0, 8, 8, 1, 0, 8, 0)",
}


def test_wrappers_link_and_throw(tmp_path):
    rocm = Path("/opt/rocm")
    if not shutil.which("g++") or not (rocm / "include/hip/hip_runtime_api.h").exists():
        pytest.skip("g++ or the HIP headers are not installed")
    text = (ROOT / "include/hymoe.hpp").read_text()
    part = text[text.index("// ---- 16-bit matrix products"):]
    assert set(re.findall(r"^inline void (\w+)\(", part, re.M)) == set(CALLS)
    body = "\n".join(f'    try {{ hymoe::{call}; std::puts("{name} -"); }} catch (const std::runtime_error &e) {{ std::printf("{name} %s\\n", e.what()); }}'
                     for name, call in CALLS.items())
    src = tmp_path / "wrappers.cpp"
    src.write_text(f'#include "hymoe.hpp"\n#include <cstdio>\n#include <stdexcept>\nint main() {{\n    hymoe::MoeDev m{{}};\n{body}\n'
                   '    std::printf("ws %zu\\n", hymoe::linear_dw_ws_bytes(0, 8, 8));\n}\n')
    exe, lib = tmp_path / "wrappers", ROOT / "hyper_amd"
    subprocess.run(["g++", "-std=c++17", "-D__HIP_PLATFORM_AMD__", f"-I{ROOT / 'include'}", f"-I{rocm}/include", str(src), "-o", str(exe), f"-L{lib}", "-lhymoe",
                    f"-L{rocm}/lib", "-lamdhip64", f"-Wl,-rpath,{lib}", f"-Wl,-rpath,{rocm}/lib"], check=True)
    out = subprocess.run([str(exe)], capture_output=True, text=True, check=True).stdout.splitlines()
    assert out[-1] == "ws 0"
    for line, name in zip(out, CALLS):
        assert line.startswith(f"{name} ") and f"hy_{name}: " in line, line
