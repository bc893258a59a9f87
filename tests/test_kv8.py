"""CPU tests of the paged 8-bit key/value cache's host side: its sizes, its
refusals, and the work lists that its kernels read (walked by a native test)."""

import os
import subprocess

import numpy as np
import pytest

import llmi_hip as H

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def shape(**kw):
    return H.Kv8Shape(**dict(dict(heads=4, kv_heads=2, head_dim=64, page_tokens=32, pages=10, slots=3), **kw))


def test_sizes():
    assert shape().sizes() == (10 * 2 * 32 * 64, 10 * 2 * 2 * 2, 3 * 2 * 4 * 16 * 64)
    big = shape(pages=1 << 20, page_tokens=256, head_dim=128)
    assert big.sizes()[0] == (1 << 20) * 2 * 256 * 128


@pytest.mark.parametrize("kw,why", [
    (dict(heads=5), "multiple of kv_heads"), (dict(heads=0), "multiple of kv_heads"), (dict(kv_heads=0), "multiple of kv_heads"),
    (dict(heads=4098), "4096"), (dict(head_dim=48), "head_dim"), (dict(head_dim=0), "head_dim"), (dict(head_dim=288), "head_dim"),
    (dict(page_tokens=0), "page_tokens"), (dict(page_tokens=24), "page_tokens"), (dict(page_tokens=1 << 17), "page_tokens"),
    (dict(pages=1 << 30, page_tokens=65536, kv_heads=4, head_dim=256), "2\\^48"), (dict(slots=1 << 30, kv_heads=4096, heads=4096), "2\\^48"),
    (dict(pages=0), "pages"), (dict(pages=1 << 31), "pages"), (dict(slots=0), "slots"), (dict(slots=1 << 31), "slots"),
])
def test_shapes_refused(kw, why):
    with pytest.raises(H.HipError, match=why):
        shape(**kw).sizes()
    with pytest.raises(H.HipError, match=why):
        H.kv8_check(shape(**kw), [0], [0], [1], [[0]])


GOOD = dict(slots=[0, 2], starts=[0, 40], counts=[30, 1], tables=[[1, 9], [0, 3]])


def test_batches_taken():
    H.kv8_check(shape(), **GOOD)
    H.kv8_check(shape(), [], [], [], np.zeros((0, 0)))
    H.kv8_check(shape(), [1], [0], [0], [[]])
    H.kv8_check(shape(), [0, 0], [32, 5], [1, 0], [[4, 5], [4, 4]])  # the second brings no tokens and reads page 4 only
    H.kv8_check(shape(), [0, 1], [32, 32], [1, 1], [[4, 5], [4, 6]])  # a shared full page


@pytest.mark.parametrize("kw,why", [
    (dict(slots=[0, 3]), "slot out of range"), (dict(slots=[-1, 0]), "slot out of range"),
    (dict(starts=[-1, 40]), "negative start"), (dict(counts=[-1, 1]), "negative count"),
    (dict(starts=[2**31 - 1, 0], counts=[1, 1]), "too many positions"),
    (dict(starts=[2**31 - 513, 0], counts=[2, 1]), "too many positions"),
    (dict(counts=[65, 1]), "too short"), (dict(tables=[[1, 9], [0, 10]]), "page out of range"),
    (dict(tables=[[-1, 9], [0, 3]]), "page out of range"),
    (dict(slots=[2, 2]), "same slot"), (dict(tables=[[1, 9], [0, 1]]), "twice"), (dict(tables=[[3, 9], [3, 3]]), "twice"),
    (dict(tables=[[1, 9], [3, 3]]), "twice"), (dict(slots=None), "without slots"),
])
def test_batches_refused(kw, why):
    with pytest.raises(H.HipError, match=why):
        H.kv8_check(shape(), **dict(GOOD, **kw))


def test_null_arrays_refused():
    lib = H.load()
    import ctypes as C

    assert lib.llmi_hip_kv8_check(C.byref(shape()), 1, None, None, None, None, 0) == 1
    assert lib.llmi_hip_kv8_check(None, 0, None, None, None, None, 0) == 1
    assert lib.llmi_hip_kv8_sizes(None, None, None, None) == 1


def test_work_lists(tmp_path):
    """tests/native/kv8_lists.cpp walks the lists of many random batches."""
    exe = str(tmp_path / "kv8_lists")
    subprocess.run(["g++", "-std=c++20", "-O1", "-g", "-fsanitize=address,undefined", "-I", os.path.join(ROOT, "include"),
                    os.path.join(ROOT, "tests", "native", "kv8_lists.cpp"), "-o", exe], check=True)
    out = subprocess.run([exe], capture_output=True, text=True)
    assert out.returncode == 0, out.stdout + out.stderr


def test_check_holds_no_more_than_the_tables():
    """A check makes no lists of work: 2^31 - 65536 new tokens need no memory a token."""
    import resource

    n = 32767
    big = shape(kv_heads=1, heads=1, head_dim=32, page_tokens=65536, pages=n, slots=1)
    table = np.arange(n, dtype=np.int32)[None]
    before = resource.getrusage(resource.RUSAGE_SELF).ru_maxrss
    H.kv8_check(big, [0], [0], [n * 65536], table)
    assert resource.getrusage(resource.RUSAGE_SELF).ru_maxrss - before < 1 << 18  # KB
