"""CPU tests of what the GPU tests of moe_kernels.py stand on: the kernels that
their calls take, and results that an h of one fp16 part misses."""

import os
import subprocess

import numpy as np
import pytest

import moe_kernels as K

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


@pytest.fixture(scope="module")
def rows(tmp_path_factory):
    exe = str(tmp_path_factory.mktemp("moe") / "moe_rows")
    subprocess.run(["g++", "-std=c++20", "-O1", "-Wall", "-Wextra", "-I", os.path.join(ROOT, "include"),
                    os.path.join(ROOT, "tests", "native", "moe_rows.cpp"), "-o", exe], check=True)

    def of(line):
        out = subprocess.run([exe], input=line, capture_output=True, text=True, check=True).stdout.split()
        return tuple(int(w) if w.isdigit() else w for w in out)
    return of


@pytest.mark.parametrize("qtype", [K.Q8_0, K.Q4_0])
def test_kernels_of_the_calls(rows, qtype):
    """A changed rule cannot move the GPU tests' calls to other kernels unseen."""
    for (count, tokens, top_k, n_in, out, per_row, _), want in K.MATMULS:
        assert rows(f"matmul {qtype} {count} {out} {n_in} {tokens * top_k} {per_row}\n") == want, (count, tokens, out)
    for (count, tokens, top_k, hidden, ffn, _), want in K.MLPS:
        assert rows(f"mlp {qtype} {qtype} {count} {hidden} {ffn} {tokens} {top_k}\n") == want, (count, tokens, hidden, ffn)
    assert {w for _, w in K.MATMULS} == {(16, "self"), (16, "tiles"), (32, "self"), (32, "tiles"), (64, "rows")}
    assert {w[:2] for _, w in K.MLPS} == {(16, 16), (16, 64), (32, 16), (32, 32), (32, 64), (64, 16), (64, 32), (64, 64), ("few",)}


@pytest.mark.parametrize("qtype,down_type", [(K.Q8_0, K.Q4_0), (K.Q4_0, K.Q8_0)])
def test_cancelling_layer(qtype, down_type):
    """Two fp16 parts of h keep the bound, one misses it by far, at every size the GPU tests use."""
    for (count, tokens, top_k, hidden, ffn, skew), _ in K.MLPS:
        rng = np.random.default_rng(ffn)
        tokens, count = min(tokens, 12), min(count, 4)
        layer = K.Cancelling(rng, qtype, down_type, count, hidden, ffn)
        ids, weights = K.draw_ids(rng, tokens, min(top_k, count), count, 0.0, skew), rng.uniform(0.5, 1, (tokens, min(top_k, count)))
        x = layer.rows(rng, tokens, hidden)
        want, bound = layer.sums(ids, weights, x)
        assert np.all(np.abs(layer.sums(ids, weights, x, 2)[0] - want) <= bound)
        assert np.all(np.abs(layer.sums(ids, weights, x, 1)[0] - want) > 8 * bound)


def test_batch_reference():
    """The results of many rows are those of one after the other."""
    rng = np.random.default_rng(1)
    (_, _, gate), (_, _, up), (_, _, down) = (K.R.matrices(rng, K.Q8_0, 2, *s) for s in ((40, 70), (40, 70), (70, 40)))
    x = rng.standard_normal((5, 70)).astype(np.float32)
    for got, want in zip(K.mlps(x, gate[1], up[1], down[1]), zip(*(K.R.mlp(r, gate[1], up[1], down[1]) for r in x))):
        assert np.allclose(got, want, rtol=1e-12, atol=0)
    for got, want in zip(K.products(x, gate[0]), zip(*(K.R.product(r, gate[0]) for r in x))):
        assert np.allclose(got, want, rtol=1e-12, atol=0)
