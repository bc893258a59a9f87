"""CPU tests of the host side of a layer of experts: calls before
llmi_hip_init, and (a native test) limits, refusals and workspace layouts."""

import ctypes as C
import os
import subprocess

import numpy as np

import llmi_hip as H
import moe_reference as R

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def test_calls_without_a_gpu():
    lib = H.load()
    n = C.c_size_t()
    assert lib.llmi_hip_moe_matmul_bytes(None, 1, 1, C.byref(n)) == 1
    assert lib.llmi_hip_moe_mlp_bytes(None, None, 1, 1, C.byref(n)) == 1
    assert lib.llmi_hip_experts_free(None) == 0


def test_plan(tmp_path):
    """tests/native/moe_plan.cpp: every refusal, and regions that never overlap."""
    exe = str(tmp_path / "moe_plan")
    subprocess.run(["g++", "-std=c++20", "-O1", "-g", "-Wall", "-Wextra", "-fsanitize=address,undefined", "-I", os.path.join(ROOT, "include"),
                    os.path.join(ROOT, "tests", "native", "moe_plan.cpp"), "-o", exe], check=True)
    out = subprocess.run([exe], capture_output=True, text=True)
    assert out.returncode == 0, out.stdout + out.stderr


def test_reference_route():
    """The 64-bit router on rows worked out by hand."""
    nan, inf = float("nan"), float("inf")
    ids, w = R.route([[0, 0, 1, 0], [-inf, nan, -inf, 2], [-inf] * 4, [inf, 0, inf, 1]], 3, True, 2.0)
    assert ids.tolist() == [[2, 0, 1], [3, -1, -1], [-1, -1, -1], [0, 2, 3]]
    e = np.exp(-1.0)
    assert np.allclose(w, [[2 / (1 + 2 * e), 2 * e / (1 + 2 * e), 2 * e / (1 + 2 * e)], [2, 0, 0], [0, 0, 0], [1, 1, 0]])
    _, w = R.route([[0, 0, 1, 0]], 1, False, 1.0)
    assert np.allclose(w, [[1 / (1 + 3 * e)]])
