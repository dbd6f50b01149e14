"""Prefix lengths of any value on the CPU: the header that the kernels take a token's
positions from, compiled for the host under the sanitizers."""
from __future__ import annotations

import os
import subprocess

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def test_prefix_lengths_of_any_value(tmp_path):
    exe = str(tmp_path / "prefix_bounds")
    subprocess.run(["g++", "-std=c++17", "-O1", "-Wall", "-Wextra", "-Werror",
                    "-fsanitize=address,undefined", "-fno-sanitize-recover=all",
                    "-I", os.path.join(ROOT, "cpp-minilamma_amd", "csrc"),
                    os.path.join(ROOT, "tests", "cpp", "prefix_bounds.cc"), "-o", exe], check=True)
    out = subprocess.run([exe], capture_output=True, text=True, timeout=120)
    assert out.returncode == 0, out.stdout + out.stderr
