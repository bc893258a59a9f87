"""CPU tests of the rules that the paged 8-bit key/value cache's host side
keeps (csrc/kv8_plan.hpp), each walked by a native program, and of the bound
that its attention is held to."""

import os
import subprocess

import numpy as np
import pytest

import kv8_precision as P

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def run_native(name, tmp_path):
    exe = str(tmp_path / name)
    subprocess.run(["g++", "-std=c++20", "-O1", "-g", "-fsanitize=address,undefined", "-I", os.path.join(ROOT, "include"),
                    os.path.join(ROOT, "tests", "native", name + ".cpp"), "-o", exe], check=True)
    out = subprocess.run([exe], capture_output=True, text=True)
    assert out.returncode == 0, out.stdout + out.stderr


def test_batches_stay_within_a_plans_limits(tmp_path):
    """A plan takes every batch of its sequences and tokens, however long the histories."""
    run_native("kv8_limits", tmp_path)


def test_captured_attention_has_room_for_shorter_drafts(tmp_path):
    """A launch captured for drafts takes every shorter one, however their rows are shared out."""
    run_native("kv8_captured", tmp_path)


def test_sequences_taken_back(tmp_path):
    """A start inside a block is allowed exactly where `open` still holds the block's earlier rows."""
    run_native("kv8_open", tmp_path)


@pytest.mark.parametrize("shape", P.SHAPES)
def test_precision_bound_has_teeth(shape):
    """The bound that the GPU's attention is held to (kv8_precision) rejects an
    attention whose q, or whose weights, have 11 bits (one fp16 part), and
    takes one with 22."""
    for largest, cut in ((8.0, "cut_q"), (1.0, "cut_w")):
        q, k, v, _, _, start = P.case(shape, largest)
        want, bound = P.attend(q, k, v, start), P.bound(q, k, v, start)
        off = [np.abs(P.attend(q, k, v, start, **{cut: bits}) - want) / bound for bits in (11, 22)]
        assert off[0].max() > 2 and off[1].max() < 0.1, (cut, off[0].max(), off[1].max())
