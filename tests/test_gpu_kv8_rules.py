"""The paged 8-bit key/value cache on the GPU (llmi_hip_kv8_*): calls that its
interface allows at the edge of what it was captured or created for, values
far from 1, and the precision that the attention states."""

import numpy as np
import pytest

import kv8_precision as P
import kv8_reference as R
import llmi_hip as H
from test_gpu_kv8 import Pool, rows_of

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("heads,kv,dim,captured", [(8, 2, 128, 5), (14, 2, 64, 3), (12, 1, 256, 4), (20, 2, 64, 6)])
def test_shorter_drafts_replayed(heads, kv, dim, captured):
    """A graph captured for drafts of `captured` tokens is replayed for every
    shorter one, with the bits of eager calls."""
    rng = np.random.default_rng(heads + captured)
    lens = [1300, 150, 40]
    pool = Pool(rng, heads, kv, dim, 32, lens)
    pool.append([0] * 3, lens, None, rows_of(rng, sum(lens), kv, dim), rows_of(rng, sum(lens), kv, dim))
    plan = H.Kv8Plan(pool.shape, 3, 3 * captured, pool.tables.size)
    size = 3 * captured * heads * dim
    qb, ob = H.DeviceBuffer(4 * size), H.DeviceBuffer(4 * size)
    plan.set(pool.slots, [30, 20, 10], [captured, 1, 0], pool.tables)
    H.synchronize()
    graph = H.Graph(lambda: plan.attention(pool.layer, qb.ptr, 0.1, ob.ptr))
    for counts in [[c, 0, 0] for c in range(1, captured + 1)] + [[c, captured, captured - c] for c in range(1, captured)]:
        starts = [n - c for n, c in zip(lens, counts)]
        q = rows_of(rng, sum(counts), heads, dim)
        want = pool.attention(starts, counts, q, 0.1)
        plan.set(pool.slots, starts, counts, pool.tables)
        for _ in range(2):
            qb.upload(q)
            ob.upload(np.full(size, 5.0, np.float32))
            graph.launch()
            H.synchronize()
            got = ob.download(np.float32).reshape(-1, heads, dim)
            assert np.array_equal(got[:len(q)], want) and (got[len(q):] == 5.0).all()


@pytest.mark.parametrize("dim,page", [(64, 32), (256, 16)])
def test_taken_back_again_and_again(dim, page):
    """Starts anywhere in the last block of either parity that was written,
    with few and many tokens from there: the cache is the quantization of the
    sequence's rows after every append."""
    rng = np.random.default_rng(dim)
    pool = Pool(rng, 2, 1, dim, page, [400])
    k, v = rows_of(rng, 400, 1, dim), rows_of(rng, 400, 1, dim)
    length, held = 0, {}  # held: parity -> (block, rows of it)
    # 40 and back to 20 (block 1), which is then the last block; its parity's 0 is gone, 16 and 0 are whole blocks.
    for start, count in ((0, 40), (20, 1), (17, 3), (16, 30), (40, 8), (33, 2), (35, 60), (95, 1), (81, 1), (82, 100), (170, 4), (0, 5), (3, 20)):
        b = start // 16
        assert start % 16 == 0 or (b % 2 in held and held[b % 2][0] == b and held[b % 2][1] >= start % 16), start
        end = start + count
        k[start:end], v[start:end] = rows_of(rng, count, 1, dim), rows_of(rng, count, 1, dim)
        pool.append([start], [count], None, k[start:end], v[start:end])
        last = (end - 1) // 16
        if b < last:
            held[(last - 1) % 2] = (last - 1, 16)
        held[last % 2] = (last, end - 16 * last)
        length = end
        gk, gv = pool.read([0], [length])
        assert np.array_equal(gk, R.quantize(k[:length]).astype(np.float32)), (start, count)
        assert np.array_equal(gv, R.quantize(v[:length]).astype(np.float32)), (start, count)


def test_model_refuses_rows_that_are_not_held():
    """A step whose start lies inside a block that its slot does not hold (any
    more) is refused before anything runs; the sequence goes on from its end."""
    import synth
    from test_gpu_kv8_model import CONFIGS

    cfg = CONFIGS["llama_4x32"]
    model = H.Model(cfg, synth.make_tensors(cfg, 5, "tiny"), H.Q8_0)
    rng = np.random.default_rng(8)
    ids = rng.integers(0, cfg["vocab_size"], 80)
    table = [[4, 1, 3, 0, 2]]
    caches = [model.new_kv8_cache(5, 16, 2, 100) for _ in range(2)]
    step = lambda c, start, n, slot=1: model.forward_kv8(c, [slot], [start], [n], table, ids[start:start + n])[0]  # noqa: E731
    one, two = caches
    step(one, 0, 40)
    step(one, 20, 1)
    for start in (5, 15, 1):  # block 0's rows have been block 2's
        with pytest.raises(H.HipError, match="not held"):
            step(one, start, 1)
    for start, slot in ((22, 1), (40, 1), (3, 0), (21, 0)):  # past the end; a slot that nothing was written under
        with pytest.raises(H.HipError, match="not held"):
            step(one, start, 1, slot)
    with pytest.raises(H.HipError, match="not held"):  # one of two sequences
        model.forward_kv8(one, [1, 0], [21, 7], [1, 1], [table[0][:2] + [0], [3, 2, 0]], [1, 2])
    # Allowed: on from the end, back inside block 1, the beginning; as if the refused steps had not been asked for.
    step(two, 0, 40)
    step(two, 20, 1)
    for start, n in ((21, 9), (17, 1), (18, 20), (33, 4), (0, 2), (1, 50)):
        assert np.array_equal(step(one, start, n), step(two, start, n)), start


@pytest.mark.parametrize("power", [-113, -100, -60, 60, 90])
@pytest.mark.parametrize("heads,kv,dim,start,count", [(4, 2, 64, 90, 1), (4, 2, 128, 90, 6), (8, 2, 64, 90, 70), (2, 1, 256, 40, 60), (4, 1, 64, 4000, 1), (4, 2, 64, 2600, 40)])
def test_attention_of_tiny_and_huge_values(heads, kv, dim, start, count, power):
    """Histories wholly of values about 2^power: a row's error counts against
    its own values, whatever kernel takes it and in however many pieces."""
    rng = np.random.default_rng(37 + dim + count)
    n = start + count
    k, v = rows_of(rng, n, kv, dim, 0.0), rows_of(rng, n, kv, dim, 0.0)
    v *= np.float32(2.0**power)
    pool = Pool(rng, heads, kv, dim, 64, [n])
    pool.append([0], [n], None, k, v)
    q = rows_of(rng, count, heads, dim, 0.0)
    got = pool.attention([start], [count], q, 0.125)
    kq, vq = R.quantize(k), R.quantize(v)
    bound = R.attend_bound(q, kq, vq, 0.125)
    want = R.attend(q, kq, vq, start, 0.125)
    assert np.abs(want).max() > 20 * bound
    assert np.abs(got - want).max() <= bound


@pytest.mark.parametrize("heads", [16, 64])  # 32 rows a key/value head, and 128
def test_attention_keeps_value_scales(heads):
    """Prompts of one block under zero keys: row t is the mean of t + 1 values,
    every weight 1.  What may be off, in roundings of 2^-24 of the largest
    value seen: the weights' and scales' digits or parts 4, the logarithm of a
    scale 2, an exponential 2, the sum's and the output's factors, their
    product and quotient 8 at most; the sums of n = t + 1 weights and of n
    products in two parts 3n.  A result this near to 2^-126 has steps of 2^-149."""
    rng = np.random.default_rng(38)
    kv, dim, count, seqs = 8, 64, 16, 12
    pool = Pool(rng, heads, kv, dim, 16, [count] * seqs)
    k, v = np.zeros((seqs * count, kv, dim), np.float32), rows_of(rng, seqs * count, kv, dim, 0.0)
    v = v.reshape(seqs, count, kv, dim) * np.exp2(rng.uniform(-113, 100, (seqs, 1, kv, 1)))
    v = v.astype(np.float32).reshape(k.shape)
    pool.append([0] * seqs, [count] * seqs, None, k, v)
    got = pool.attention([0] * seqs, [count] * seqs, rows_of(rng, seqs * count, heads, dim, 0.0), 0.125)
    got = got.reshape(seqs, count, kv, heads // kv, dim).astype(np.float64)
    n = np.arange(1, count + 1)[:, None, None, None]
    for i in range(seqs):
        vq = R.quantize(v[i * count:(i + 1) * count])[:, :, None]
        want = np.cumsum(vq, 0) / n
        seen = np.maximum.accumulate(np.abs(vq).max(-1, keepdims=True), 0)
        off = np.abs(got[i] - want)
        assert (off <= seen * (16 + 3 * n) * 2.0**-24 + 2.0**-149).all(), (i, (off / seen).max() * 2**24)


def test_as_many_sequences_as_a_plan_takes():
    """2^20 sequences that read the same page, of 8 heads each: more workgroups
    than a launch may have (2^32 threads), so each takes several units."""
    rng = np.random.default_rng(39)
    kv, dim, seqs, some = 8, 32, 1 << 20, 1 << 12
    pool = Pool(rng, kv, kv, dim, 16, [3])
    k, v = rows_of(rng, 3, kv, dim), rows_of(rng, 3, kv, dim)
    pool.append([0], [3], None, k, v)
    plan = H.Kv8Plan(pool.shape, seqs, seqs, seqs)
    plan.set(None, np.full(seqs, 2), np.ones(seqs), np.broadcast_to(pool.tables, (seqs, 1)))
    q = rows_of(rng, some, kv, dim, 0.0)
    qb = H.DeviceBuffer.from_array(np.tile(q.reshape(1, -1), (seqs // some, 1)))
    ob = H.DeviceBuffer.from_array(np.full(seqs * kv * dim, np.nan, np.float32))
    plan.attention(pool.layer, qb.ptr, 0.2, ob.ptr)
    H.synchronize()
    got = ob.download(np.float32).reshape(seqs // some, some, kv, dim)
    kq, vq = R.quantize(k), R.quantize(v)
    p = np.exp(0.2 * np.einsum("nhd,jhd->nhj", q.astype(np.float64), kq))
    want = np.einsum("nhj,jhd->nhd", p / p.sum(-1, keepdims=True), vq)
    assert np.abs(got[0] - want).max() <= R.attend_bound(q, kq, vq, 0.2)
    assert all(np.array_equal(x, got[0]) for x in got[1:])


@pytest.mark.parametrize("shape", P.SHAPES)
@pytest.mark.parametrize("largest", [1.0, 8.0])
def test_attention_keeps_22_bits(shape, largest):
    """q and the weights with fewer bits than promised would show (see kv8_precision)."""
    heads, kv, dim, start, count = shape
    q, kq, vq, k, v, _ = P.case(shape, largest)
    pool = Pool(np.random.default_rng(40), heads, kv, dim, 32, [start + count])
    pool.append([0], [start + count], None, k, v)
    got = pool.attention([start], [count], q, P.SCALE)
    off = np.abs(got - P.attend(q, kq, vq, start)) / P.bound(q, kq, vq, start)
    assert off.max() <= 1, off.max()


def test_model_steps_of_many_tokens():
    """65535 tokens in one step; one more is refused before anything runs, and
    the sequences go on from where they were."""
    import synth
    from test_gpu_kv8_model import CONFIGS

    cfg = CONFIGS["llama_4x32"]
    model = H.Model(cfg, synth.make_tensors(cfg, 6, "tiny"), H.Q8_0)
    rng = np.random.default_rng(41)
    n = 257
    cache = model.new_kv8_cache(16 * n, 16, n, 70000)
    tables = rng.permutation(16 * n).reshape(n, 16)
    ids = rng.integers(0, cfg["vocab_size"], (n, 256))
    counts = [256] * 255 + [255, 0]
    first = model.forward_kv8(cache, range(n), [0] * n, counts, tables, np.concatenate([ids[i, :c] for i, c in enumerate(counts)]))
    with pytest.raises(H.HipError, match="65535 tokens"):
        model.forward_kv8(cache, range(n), [0] * n, [256] * 255 + [255, 1], tables, np.concatenate([ids[:255].reshape(-1), ids[255, :255], ids[256, :1]]))
    then = model.forward_kv8(cache, [255], [255], [1], tables[255:256], ids[255, 255:])
    alone = model.new_kv8_cache(16, 16, 1, 256)
    for got, i, c in ((first, 0, 256), (first, 254, 256), (first, 255, 255)):
        want = model.forward_kv8(alone, [0], [0], [c], [range(16)], ids[i, :c])[0]
        assert np.abs(got[i] - want).max() <= 1e-4 * np.abs(want).max()  # the order of fp32 sums, as in test_alone_and_together_agree
    want = model.forward_kv8(alone, [0], [255], [1], [range(16)], ids[255, 255:])[0]
    assert np.abs(then[0] - want).max() <= 1e-4 * np.abs(want).max()
