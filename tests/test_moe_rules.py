"""CPU tests of rules that every call of a layer of experts checks on the host."""

import os
import subprocess

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def test_overlap(tmp_path):
    """tests/native/moe_overlap.cpp: operands that meet, byte by byte."""
    exe = str(tmp_path / "moe_overlap")
    subprocess.run(["g++", "-std=c++20", "-O1", "-g", "-Wall", "-Wextra", "-fsanitize=address,undefined", "-I", os.path.join(ROOT, "include"),
                    os.path.join(ROOT, "tests", "native", "moe_overlap.cpp"), "-o", exe], check=True)
    out = subprocess.run([exe], capture_output=True, text=True)
    assert out.returncode == 0, out.stdout + out.stderr
