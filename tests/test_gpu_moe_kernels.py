"""Every kernel of the experts' products on the GPU: each size of a group of
rows, both types, one and many steps of inputs (the calls of moe_kernels.py),
and the second fp16 part of the results between an MLP's products."""

import numpy as np
import pytest

import llmi_hip as H
import moe_kernels as K
import test_gpu_moe as G
from test_oracle_gguf import GGUF_Q4_0, GGUF_Q8_0

pytestmark = pytest.mark.gpu

TYPES = [H.Q8_0, H.Q4_0]


def names(calls):
    return ["-".join(map(str, call)) for call, _ in calls]


@pytest.mark.parametrize("qtype", TYPES)
@pytest.mark.parametrize("call", [c for c, _ in K.MATMULS], ids=names(K.MATMULS))
def test_matmul_kernels(qtype, call):
    count, tokens, top_k, n_in, out, per_row, skew = call
    rng = np.random.default_rng(n_in * 13 + out)
    experts, values = G.make(rng, qtype, count, out, n_in)
    ids = K.draw_ids(rng, tokens, top_k, count, 0.05, skew)
    x = (rng.standard_normal((ids.size // per_row, n_in)) * np.exp(rng.standard_normal(n_in))).astype(np.float32)
    y = G.run_matmul(experts, ids, x, per_row, n_in + 1, out + 3)
    flat = ids.reshape(-1)
    assert (y[flat < 0] == G.GUARD).all()
    for e in range(count):
        s = np.nonzero(flat == e)[0]
        if len(s):
            want, bound = K.products(x[s // per_row], values[e])
            assert np.all(np.abs(y[s] - want) <= bound), e


@pytest.mark.parametrize("qtype,down_type", [(a, b) for a in TYPES for b in TYPES])
@pytest.mark.parametrize("call", [c for c, _ in K.MLPS], ids=names(K.MLPS))
def test_mlp_kernels(qtype, down_type, call):
    count, tokens, top_k, hidden, ffn, skew = call
    rng = np.random.default_rng(hidden * 17 + ffn)
    layer = G.Layer(rng, qtype, down_type, count, hidden, ffn)
    ids = K.draw_ids(rng, tokens, top_k, count, 0.05 if tokens > 2 else 0.0, skew)
    weights = rng.random((tokens, top_k)).astype(np.float32)
    x = rng.standard_normal((tokens, hidden)).astype(np.float32)
    want, bound = K.sums(ids, weights, x, layer.vg, layer.vu, layer.vd)
    assert np.all(np.abs(layer.run(ids, weights, x, pad=1) - want) <= bound)


class Loaded(G.Layer):
    """A layer of given planar matrices."""

    def __init__(self, matrices, types):
        for (name, (codes, scales, values)), qtype in zip(matrices.items(), types):
            d, s = G.dev(codes), G.dev(scales)
            setattr(self, name, H.Experts.upload_dev(d.ptr, s.ptr, *values.shape, qtype))


@pytest.mark.parametrize("qtype,down_type", [(a, b) for a in TYPES for b in TYPES])
@pytest.mark.parametrize("call", [c for c, _ in K.MLPS], ids=names(K.MLPS))
def test_second_part_between_the_products(qtype, down_type, call):
    """Results that an h rounded to fp16 would make 0."""
    count, tokens, top_k, hidden, ffn, skew = call
    rng = np.random.default_rng(hidden * 19 + ffn)
    plain = K.Cancelling(rng, qtype, down_type, count, hidden, ffn)
    layer = Loaded(plain.matrices, (qtype, qtype, down_type))
    ids = K.draw_ids(rng, tokens, top_k, count, 0.05 if tokens > 2 else 0.0, skew)
    weights = rng.uniform(0.5, 1, (tokens, top_k)).astype(np.float32)
    x = plain.rows(rng, tokens, hidden)
    want, bound = plain.sums(ids, weights, x)
    y = layer.run(ids, weights, x)
    assert np.all(np.abs(y - want) <= bound), (np.abs(y - want) / np.maximum(bound, 1e-30)).max()


@pytest.mark.parametrize("qtype", TYPES)
@pytest.mark.parametrize("out,n_in", [(37, 96), (64, 256), (5, 32)])
def test_experts_from_gguf(qtype, out, n_in):
    """Experts of weights that GGUF blocks were loaded into: the bits of planar codes and scales."""
    rng = np.random.default_rng(out + n_in)
    count, blocks = 3, n_in // 32
    codes = rng.integers(-8 if qtype == H.Q4_0 else -127, 8 if qtype == H.Q4_0 else 128, (count, out, blocks, 32), dtype=np.int8)
    scales = (rng.random((count, out, blocks)) + 0.5).astype(np.float16)
    if qtype == H.Q8_0:
        packed = codes.view(np.uint8)
    else:  # element i in the low half of byte i, i + 16 in the high one
        packed = (codes[..., :16] + 8).astype(np.uint8) | (codes[..., 16:] + 8).astype(np.uint8) << 4
    raw = np.concatenate([scales[..., None].view(np.uint8), packed], -1)
    gguf = GGUF_Q8_0 if qtype == H.Q8_0 else GGUF_Q4_0
    a = H.Experts.from_weights([H.Weight.from_gguf(raw[e].reshape(-1), out, n_in, gguf) for e in range(count)])
    flat = codes.reshape(count, out, n_in)
    d, s = G.dev(K.planar(flat, qtype)), G.dev(scales.astype(np.float32))
    b = H.Experts.upload_dev(d.ptr, s.ptr, count, out, n_in, qtype)
    values = flat * np.repeat(scales.astype(np.float64), 32, -1)
    ids = np.arange(130, dtype=np.int32) % 4 - 1
    for slots in (9, 130):
        x = rng.standard_normal((slots, n_in)).astype(np.float32)
        ya, yb = G.run_matmul(a, ids[:slots], x, 1), G.run_matmul(b, ids[:slots], x, 1)
        assert np.array_equal(ya.view(np.uint32), yb.view(np.uint32))
        G.check_matmul(ya, ids[:slots], x, 1, values)


@pytest.mark.parametrize("qtype", TYPES)
@pytest.mark.parametrize("down_size,weight", [(2.0**-7, 1.0), (2.0**6, 2.0**-18)])
@pytest.mark.parametrize("call", [c for c, _ in K.MLPS], ids=names(K.MLPS))
def test_mlp_small_results(qtype, call, down_size, weight):
    """Results of about 2^-113 between the products, whose scales and weights take them further down."""
    count, tokens, top_k, hidden, ffn, skew = call
    rng = np.random.default_rng(hidden * 23 + ffn)
    mats = {n: K.R.matrices(rng, qtype, count, *s, 0.3) for n, s in (("gate", (ffn, hidden)), ("up", (ffn, hidden)), ("down", (hidden, ffn)))}
    codes, scales, values = mats["down"]
    mats["down"] = codes, scales * np.float32(down_size), values * down_size
    layer = Loaded(mats, (qtype,) * 3)
    ids = K.draw_ids(rng, tokens, top_k, count, 0.0, skew)
    weights = (rng.uniform(0.5, 1, (tokens, top_k)) * weight).astype(np.float32)
    x = (rng.standard_normal((tokens, hidden)) * 2.0**-56).astype(np.float32)
    want, bound = K.sums(ids, weights, x, *(mats[n][2] for n in ("gate", "up", "down")))
    # Below the normal numbers a rounding is 2^-150: of every element of h, and
    # of every addition over blocks, waves and choices.
    steps = -(-ffn // 32) + 32 + 2 * top_k
    bound += top_k * weight * np.abs(mats["down"][2]).sum(2).max() * 2.0**-149 + steps * 2.0**-149
    assert np.all(np.abs(layer.run(ids, weights, x) - want) <= bound), (np.abs(layer.run(ids, weights, x) - want) / bound).max()


@pytest.mark.parametrize("qtype", TYPES)
@pytest.mark.parametrize("size,x_size", [(2.0**79, 2.0**-70), (2.0**-110, 2.0**100), (-(2.0**-30), 2.0**-90)])
@pytest.mark.parametrize("call", [(2, 1, 2, 100, 40, 2, 1.0), (2, 9, 1, 300, 70, 1, 1.0)] + [K.MATMULS[i][0] for i in (2, 5, 8, 13)])
def test_matmul_scales_of_any_size(qtype, size, x_size, call):
    """Scales up to 2^80 with rows that bring the results back, tiny and negative ones."""
    count, tokens, top_k, n_in, out, per_row, skew = call
    rng = np.random.default_rng(n_in * 29 + out)
    codes, scales, values = K.R.matrices(rng, qtype, count, out, n_in, 0.0)
    scales, by = np.full_like(scales, size), size / scales[0, 0, 0].astype(np.float64)
    d, s = G.dev(codes), G.dev(scales)
    experts = H.Experts.upload_dev(d.ptr, s.ptr, count, out, n_in, qtype)
    ids = K.draw_ids(rng, tokens, top_k, count, 0.0, skew)
    x = (rng.standard_normal((ids.size // per_row, n_in)) * x_size).astype(np.float32)
    y = G.run_matmul(experts, ids, x, per_row)
    flat = ids.reshape(-1)
    for e in range(count):
        r = np.nonzero(flat == e)[0]
        if len(r):
            want, bound = K.products(x[r // per_row], values[e] * by)
            assert np.all(np.abs(y[r] - want) <= bound + 2.0**-149 * (n_in / 32 + 16)), e


@pytest.mark.parametrize("qtype", TYPES)
@pytest.mark.parametrize("down_size", [2.0**80, 2.0**-100])
@pytest.mark.parametrize("call", [K.MLPS[i][0] for i in (0, 2, 6, 11, 13, 16, 17)])
def test_mlp_scales_of_any_size(qtype, down_size, call):
    """The same for an MLP's second product."""
    count, tokens, top_k, hidden, ffn, skew = call
    rng = np.random.default_rng(hidden * 31 + ffn)
    mats = {n: K.R.matrices(rng, qtype, count, *s, 0.0) for n, s in (("gate", (ffn, hidden)), ("up", (ffn, hidden)), ("down", (hidden, ffn)))}
    codes, scales, values = mats["down"]
    mats["down"] = codes, np.full_like(scales, down_size), values * (down_size / scales[0, 0, 0].astype(np.float64))
    layer = Loaded(mats, (qtype,) * 3)
    ids = K.draw_ids(rng, tokens, top_k, count, 0.0, skew)
    weights = rng.random((tokens, top_k)).astype(np.float32)
    x = rng.standard_normal((tokens, hidden)).astype(np.float32)
    want, bound = K.sums(ids, weights, x, *(mats[n][2] for n in ("gate", "up", "down")))
    assert np.all(np.abs(layer.run(ids, weights, x) - want) <= bound)
