"""CPU tests of rules that every call of a layer of experts checks on the host."""

import os
import re
import subprocess

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def test_overlap(tmp_path):
    """tests/native/moe_overlap.cpp: operands that meet, byte by byte."""
    exe = str(tmp_path / "moe_overlap")
    subprocess.run(["g++", "-std=c++20", "-O1", "-g", "-Wall", "-Wextra", "-fsanitize=address,undefined", "-I", os.path.join(ROOT, "include"),
                    os.path.join(ROOT, "tests", "native", "moe_overlap.cpp"), "-o", exe], check=True)
    out = subprocess.run([exe], capture_output=True, text=True)
    assert out.returncode == 0, out.stdout + out.stderr


def test_assembly_names_the_registers_it_writes():
    """The compiler keeps nothing in a special register that an asm statement sets."""
    csrc = os.path.join(ROOT, "llm-inference-cpp_amd", "csrc")
    writes = 0
    for name in sorted(os.listdir(csrc)):
        with open(os.path.join(csrc, name)) as f:
            for statement in re.findall(r"\basm\b[^;]*;", f.read()):
                for reg in re.findall(r"\bs_mov_b32 (m0|exec|vcc)\b", statement):
                    writes += 1
                    assert f'"{reg}"' in statement.rsplit(":", 1)[-1], (name, statement)
    assert writes == 2
