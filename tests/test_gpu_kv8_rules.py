"""The paged 8-bit key/value cache on the GPU (llmi_hip_kv8_*): calls that its
interface allows at the edge of what it was captured or created for."""

import numpy as np
import pytest

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
