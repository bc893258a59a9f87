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
