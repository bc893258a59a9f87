"""CPU tests of the rules that the paged 8-bit key/value cache's host side
keeps (csrc/kv8_plan.hpp), each walked by a native program."""

import os
import subprocess

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
