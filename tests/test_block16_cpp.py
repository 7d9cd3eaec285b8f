"""include/hymoe.hpp's wrappers of the norms, of routing with groups and of the low-rank adapters: a program that calls each links
against the library, and what the C entry refuses arrives as an exception with its message."""
import re
import shutil
import subprocess
from pathlib import Path

import pytest

ROOT = Path(__file__).resolve().parents[1]
CALLS = {
    "norm": "norm(9, 0, 0, 8, 0, 0, 0, 0, 0, 0, 0.0f, 1, 8, 0, 0, 8, 0, 0, 0, 0, 0)",
    "norm_bwd": "norm_bwd(9, 0, 0, 8, 0, 0, 8, 0, 0, 0, 0, 0, 1, 8, 0, 8, 0, 0, false, 0, 0, 0)",
    "moe_route_groups": "moe_route_groups(0, 8, 8, 0, 9, 1, 1, 1, 2, true, 1.0f, 0, 0, 1, 0)",
    "moe_route_groups_bwd": "moe_route_groups_bwd(0, 8, 8, 9, 0, 2, true, 1.0f, 0, 0, 0, 8, 1, 0)",
    "lora": "lora(7, 0, 0, 0, 1, 4, 8, 8, 0, 8, 1, 0, 0, 0, 0, 0, 8, 0, 0, 0)",
}


def test_wrappers_link_and_throw(tmp_path):
    rocm = Path("/opt/rocm")
    if not shutil.which("g++") or not (rocm / "include/hip/hip_runtime_api.h").exists():
        pytest.skip("g++ or the HIP headers are not installed")
    text = (ROOT / "include/hymoe.hpp").read_text()
    part = text[text.index("// ---- around the 16-bit products"):text.index("// ---- 16-bit matrix products")]
    assert set(re.findall(r"^inline void (\w+)\(", part, re.M)) == set(CALLS)
    body = "\n".join(f'    try {{ hymoe::{call}; std::puts("{name} -"); }} catch (const std::runtime_error &e) {{ std::printf("{name} %s\\n", e.what()); }}'
                     for name, call in CALLS.items())
    src = tmp_path / "wrappers.cpp"
    src.write_text(f'#include "hymoe.hpp"\n#include <cstdio>\n#include <stdexcept>\nint main() {{\n{body}\n'
                   '    std::printf("ws %zu %zu\\n", hymoe::norm_bwd_ws_bytes(1, 8), hymoe::lora_ws_bytes(3, 4, 8));\n}\n')
    exe, lib = tmp_path / "wrappers", ROOT / "hyper_amd"
    subprocess.run(["g++", "-std=c++17", "-D__HIP_PLATFORM_AMD__", f"-I{ROOT / 'include'}", f"-I{rocm}/include", str(src), "-o", str(exe), f"-L{lib}", "-lhymoe",
                    f"-L{rocm}/lib", "-lamdhip64", f"-Wl,-rpath,{lib}", f"-Wl,-rpath,{rocm}/lib"], check=True)
    out = subprocess.run([str(exe)], capture_output=True, text=True, check=True).stdout.splitlines()
    assert out[-1] == "ws 0 48"
    for line, name in zip(out, CALLS):
        assert line.startswith(f"{name} ") and f"hy_{name}: " in line, line
