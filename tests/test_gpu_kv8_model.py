"""llmi_hip_model_forward_kv8: sequences run together over a model's paged
8-bit cache, against the model computed in 64 bits with the same cache
(tests/kv8_reference.py)."""

import numpy as np
import pytest

import kv8_reference as R
import llmi_hip as H
import synth

pytestmark = pytest.mark.gpu

CONFIGS = {
    "llama_4x32": dict(arch=0, vocab_size=64, hidden_size=128, intermediate_size=96, num_layers=2, num_heads=4, num_kv_heads=2,
                       max_position_embeddings=256, rms_norm_eps=1e-5, rope_theta=10000.0, tie_word_embeddings=1, qkv_bias=0),
    "qwen_3x64": dict(arch=1, vocab_size=50, hidden_size=192, intermediate_size=128, num_layers=3, num_heads=3, num_kv_heads=1,
                      max_position_embeddings=200, rms_norm_eps=1e-6, rope_theta=100000.0, tie_word_embeddings=0, qkv_bias=1),
}


def weights(cfg, qtype):
    """(host tensors for the model, the values its matrices hold in 64 bits)."""
    specs, tensors = synth.tensor_specs(cfg), synth.make_tensors(cfg, 11, "tiny")
    values = []
    for (_, shape, kind), t in zip(specs, tensors):
        if kind == "matrix" and qtype != H.F32:
            w = H.Weight.quantize(t, shape[0], shape[1], qtype)
            values.append(np.stack([w.dequantize_row(r) for r in range(shape[0])]).astype(np.float64))
            w.free()
        else:
            values.append(t.reshape(shape).astype(np.float64))
    return tensors, values


class Reference:
    """The model in 64 bits; one sequence's keys and values as the cache holds them."""

    def __init__(self, cfg, values):
        self.cfg, self.it = cfg, values
        self.hd = cfg["hidden_size"] // cfg["num_heads"]
        half = np.arange(0, self.hd, 2, dtype=np.float32) / np.float32(self.hd)
        freq = (1.0 / cfg["rope_theta"] ** half.astype(np.float64)).astype(np.float32)
        angle = (np.arange(cfg["max_position_embeddings"], dtype=np.float32)[:, None] * freq).astype(np.float64)
        self.cos, self.sin = np.cos(angle).astype(np.float32), np.sin(angle).astype(np.float32)

    def run(self, ids, kept):
        """Logits of the last of `ids`, after len(kept[0][0]) earlier positions;
        kept: per layer (k, v) rows before they are quantized, extended in place."""
        cfg, hd = self.cfg, self.hd
        norm = lambda x, w: x / np.sqrt((x * x).mean(-1, keepdims=True) + cfg["rms_norm_eps"]) * w  # noqa: E731
        it = iter(self.it)
        embed = next(it)
        x, start = embed[ids], len(kept[0][0])
        at = slice(start, start + len(ids))
        for layer in range(cfg["num_layers"]):
            h = norm(x, next(it))
            q, k, v = (h @ next(it).T for _ in range(3))
            if cfg["qkv_bias"]:
                q, k, v = (y + next(it) for y in (q, k, v))
            q, k, v = (y.reshape(len(ids), -1, hd) for y in (q, k, v))
            q, k = (R.turn(y, None, 0, self.cos[at][:, None], self.sin[at][:, None]) for y in (q, k))
            kept[layer] = tuple(np.concatenate([a, b.astype(np.float32)]) for a, b in zip(kept[layer], (k, v)))
            kq, vq = (R.quantize(y) for y in kept[layer])
            att = R.attend(q, kq, vq, start, hd ** -0.5)
            x = x + att.reshape(len(ids), -1) @ next(it).T
            h = norm(x, next(it))
            g, u = h @ next(it).T, h @ next(it).T
            x = x + (g / (1 + np.exp(-g)) * u) @ next(it).T
        last = norm(x[-1], next(it))
        return (embed if cfg["tie_word_embeddings"] else next(it)) @ last

    def empty(self):
        return [(np.zeros((0, self.cfg["num_kv_heads"], self.hd), np.float32),) * 2 for _ in range(self.cfg["num_layers"])]


@pytest.mark.parametrize("name,qtype,page", [("llama_4x32", H.F32, 16), ("llama_4x32", H.Q8_0, 32), ("qwen_3x64", H.Q4_0, 48), ("qwen_3x64", H.F32, 16)])
def test_steps_of_several_sequences(name, qtype, page):
    """Prompts, pieces of prompts and single tokens side by side; a sequence
    that ends and one that begins in its slot and pages.

    The model's activations are fp32 and the reference's 64-bit, so a key or
    value that lies within some 1e-6 of a rounding border may get the next
    code: one of dim values off by 1/127 of its block's largest, weighted by
    its position's probability.  Logits may differ by a few such steps over
    the number of summed terms (dim >= 32): 1/127 / 32 * 8 = 2e-3 of the largest."""
    cfg = CONFIGS[name]
    rng = np.random.default_rng(len(name) + qtype)
    tensors, values = weights(cfg, qtype)
    ref, model = Reference(cfg, values), H.Model(cfg, tensors, qtype)
    slots, width = 3, -(-cfg["max_position_embeddings"] // page)
    cache = model.new_kv8_cache(slots * width, page, slots, 256)
    pages = rng.permutation(slots * width).reshape(slots, width)
    state = [[ref.empty(), 0] for _ in range(slots)]
    steps = [(20, 33, 1), (1, 7, 15), (1, 1, 0), (5, 1, 1), (0, 0, 1), (1, 40, 1)] + [(1, 1, 1)] * 3
    for n, counts in enumerate(steps):
        if n == 4:
            state[1] = [ref.empty(), 0]  # the second sequence ends; another takes its slot
        ids = [rng.integers(0, cfg["vocab_size"], c) for c in counts]
        got = model.forward_kv8(cache, range(slots), [s[1] for s in state], counts, pages, np.concatenate(ids))
        row = 0
        for s, x in zip(state, ids):
            if len(x) == 0:
                continue
            want = ref.run(x, s[0])
            s[1] += len(x)
            assert np.abs(got[row] - want).max() <= 2e-3 * np.abs(want).max(), (n, row)
            row += 1
        assert row == len(got)
    cache.free()
    model.free()


def test_alone_and_together_agree():
    """A sequence's logits do not depend on its company beyond the order of
    fp32 sums (histories are split by the size of the batch): 2^-24 a sum of
    some hundred terms, through three layers."""
    cfg = CONFIGS["qwen_3x64"]
    tensors, _ = weights(cfg, H.Q8_0)
    model = H.Model(cfg, tensors, H.Q8_0)
    rng = np.random.default_rng(3)
    n, width = 4, 13
    ids = [rng.integers(0, cfg["vocab_size"], 120 + 7 * i) for i in range(n)]
    pages = np.arange(n * width).reshape(n, width)
    both = model.new_kv8_cache(n * width, 16, n, 600)
    first = model.forward_kv8(both, range(n), [0] * n, [len(x) for x in ids], pages, np.concatenate(ids))
    then = model.forward_kv8(both, range(n), [len(x) for x in ids], [1] * n, pages, [5] * n)
    for i in range(n):
        one = model.new_kv8_cache(width, 16, 1, 200)
        a = model.forward_kv8(one, [0], [0], [len(ids[i])], [range(width)], ids[i])
        b = model.forward_kv8(one, [0], [len(ids[i])], [1], [range(width)], [5])
        for alone, got in ((a[0], first[i]), (b[0], then[i])):
            assert np.abs(alone - got).max() <= 1e-4 * np.abs(got).max()


def test_fp32_and_8bit_caches_stay_apart():
    """The exact calls give the same bits before and after steps over the 8-bit cache."""
    cfg = CONFIGS["llama_4x32"]
    tensors, _ = weights(cfg, H.Q8_0)
    model = H.Model(cfg, tensors, H.Q8_0)
    ids = np.arange(40) % cfg["vocab_size"]
    before = model.forward(ids)
    cache = model.new_kv8_cache(8, 16, 2, 64)
    model.forward_kv8(cache, [0, 1], [0, 0], [40, 3], [[0, 1, 2], [3, 4, 5]], np.concatenate([ids, ids[:3]]))
    assert np.array_equal(before, model.forward(ids))
    assert np.array_equal(model.generate_greedy(ids[:5], 8), model.generate_greedy(ids[:5], 8))


def test_refusals():
    cfg = CONFIGS["llama_4x32"]
    tensors, _ = weights(cfg, H.F32)
    model, other = H.Model(cfg, tensors, H.F32), H.Model(cfg, tensors, H.F32)
    no = lambda match: pytest.raises(H.HipError, match=match)  # noqa: E731
    for args, match in (((0, 16, 1, 8), "pages"), ((4, 24, 1, 8), "page_tokens"), ((4, 16, 0, 8), "slots"), ((4, 16, 1, 0), "max_tokens")):
        with no(match):
            model.new_kv8_cache(*args)
    odd = dict(cfg, hidden_size=48 * 4, num_heads=4)  # head size 48
    small = H.Model(odd, synth.make_tensors(odd, 1, "tiny"), H.F32)
    with no("head_dim"):
        small.new_kv8_cache(4, 16, 1, 8)
    cache = model.new_kv8_cache(20, 16, 2, 24)
    step = lambda m, slots, starts, counts, tables, toks: m.forward_kv8(cache, slots, starts, counts, tables, toks)  # noqa: E731
    with no("not created by this model"):
        step(other, [0], [0], [1], [[0]], [1])
    with no("no tokens"):
        step(model, [0], [0], [0], [[0]], [])
    with no("out of range"):
        step(model, [0], [0], [2], [[0]], [1, 64])
    with no("out of range"):
        step(model, [0], [0], [1], [[0]], [-1])
    with no("page out of range"):
        step(model, [0], [0], [1], [[20]], [1])
    with no("slot out of range"):
        step(model, [2], [0], [1], [[0]], [1])
    with no("same slot"):
        step(model, [0, 0], [0, 0], [1, 1], [[0], [1]], [1, 1])
    with no("twice"):
        step(model, [0, 1], [0, 0], [1, 1], [[1], [1]], [1, 1])
    with no("too short"):
        step(model, [0], [16], [1], [[0]], [1])
    with no("more tokens"):
        step(model, [0], [0], [25], [[0, 1]], [1] * 25)
    with no("context"):
        step(model, [0], [256], [1], [range(17)], [1])
    with pytest.raises(ValueError):
        step(model, [0], [0], [2], [[0]], [1])
    assert np.isfinite(step(model, [0], [0], [3], [[0]], [1, 2, 3])).all()


def test_a_cache_that_does_not_fit_leaves_no_error_behind():
    cfg = CONFIGS["llama_4x32"]
    tensors, _ = weights(cfg, H.F32)
    model = H.Model(cfg, tensors, H.F32)
    cache = model.new_kv8_cache(4, 16, 1, 8)
    want = model.forward_kv8(cache, [0], [0], [3], [[1]], [5, 6, 7])
    with pytest.raises(H.HipError, match="out of memory"):
        model.new_kv8_cache(2**31 - 1, 16, 1, 8)  # 4 TiB of keys
    assert np.array_equal(model.forward_kv8(cache, [0], [0], [3], [[1]], [5, 6, 7]), want)
