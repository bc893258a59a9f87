"""The paged 8-bit key/value cache on the GPU (llmi_hip_kv8_*): append, read
and attention against tests/kv8_reference.py, alone and together."""

import numpy as np
import pytest

import kv8_reference as R
import llmi_hip as H

pytestmark = pytest.mark.gpu

EPS = 1e-5


class Pool:
    """A device cache for sequences of up to `lens` positions, filled with garbage."""

    def __init__(self, rng, heads, kv, dim, page, lens, spare=3):
        self.tables, pages = R.tables(rng, lens, page, spare)
        self.slots = rng.permutation(len(lens)).astype(np.int32)
        self.shape = H.Kv8Shape(heads, kv, dim, page, pages, max(len(lens), 1))
        code, scale, opened = self.shape.sizes()
        junk = rng.integers(-128, 128, code, dtype=np.int8)
        self.bufs = [H.DeviceBuffer.from_array(junk), H.DeviceBuffer.from_array(junk[::-1].copy()),
                     H.DeviceBuffer.from_array(np.full(scale, np.nan, np.float32)),
                     H.DeviceBuffer.from_array(np.full(opened, np.nan, np.float32))]
        self.layer = H.Kv8Layer(*(b.ptr for b in self.bufs))
        self.heads, self.kv, self.dim = heads, kv, dim

    def plan(self, starts, counts, max_tokens=None, rows=None):
        rows = list(range(len(starts))) if rows is None else rows
        p = H.Kv8Plan(self.shape, max(len(rows), 1), max_tokens or max(int(np.sum(counts)), 1), self.tables.size)
        p.set(self.slots[rows], starts, counts, self.tables[rows])
        return p

    def append(self, starts, counts, q, k, v, rows=None, **more):
        """Appends host rows; returns q as it comes back (None without q)."""
        p = self.plan(starts, counts, rows=rows)
        kb, vb = (H.DeviceBuffer.from_array(a.astype(np.float32)) for a in (k, v))
        qb = None if q is None else H.DeviceBuffer.from_array(q.astype(np.float32))
        ob = None if q is None else H.DeviceBuffer(q.size * 4)
        keep, args = [], dict(more)
        for name in ("q_norm", "k_norm", "cos", "sin"):
            if args.get(name) is not None:
                if name == "cos":
                    args["positions"] = len(args["cos"])
                keep.append(H.DeviceBuffer.from_array(args[name]))
                args[name] = keep[-1].ptr
        p.append(self.layer, None if q is None else qb.ptr, kb.ptr, vb.ptr, None if q is None else ob.ptr, **args)
        H.synchronize()
        return None if q is None else ob.download(np.float32).reshape(q.shape)

    def read(self, starts, counts, rows=None):
        n = int(np.sum(counts))
        if n == 0:
            return (np.zeros((0, self.kv, self.dim), np.float32),) * 2
        kb, vb = (H.DeviceBuffer(n * self.kv * self.dim * 4) for _ in range(2))
        p = self.plan(starts, counts, rows=rows)
        p.read(self.layer, kb.ptr, vb.ptr)
        H.synchronize()
        return [b.download(np.float32).reshape(n, self.kv, self.dim) for b in (kb, vb)]

    def attention(self, starts, counts, q, scale, rows=None):
        p = self.plan(starts, counts, rows=rows)
        qb, ob = H.DeviceBuffer.from_array(q.astype(np.float32)), H.DeviceBuffer(q.size * 4)
        p.attention(self.layer, qb.ptr, scale, ob.ptr)
        H.synchronize()
        return ob.download(np.float32).reshape(q.shape)


def rows_of(rng, n, heads, dim, spread=1.0):
    return (rng.standard_normal((n, heads, dim)) * np.exp(rng.standard_normal((n, heads, 1)) * spread)).astype(np.float32)


def once(got, want):
    """One rounding of a value computed in 64 bits."""
    want = np.asarray(want, dtype=np.float64)
    assert np.all(np.abs(got - want) <= np.abs(want) * (2.0**-24 * 1.0001) + 1e-13 * np.abs(want).max(-1, keepdims=True))


APPENDS = [
    # heads, kv, dim, page, starts, counts, norm, rotation
    (4, 2, 64, 16, [0], [1], False, True),
    (9, 3, 64, 64, [0, 0, 0], [1, 16, 17], False, True),
    (14, 2, 64, 32, [0, 0], [40, 0], True, True),
    (8, 8, 32, 48, [0, 0, 0, 0], [15, 31, 33, 2], True, False),
    (6, 2, 96, 16, [0, 0], [50, 7], True, True),
    (5, 1, 128, 128, [0, 0], [130, 1], False, False),
    (4, 4, 160, 32, [0], [35], True, True),
    (2, 1, 224, 16, [0], [19], False, True),
    (3, 1, 256, 64, [0, 0], [66, 16], True, True),
]


@pytest.mark.parametrize("heads,kv,dim,page,starts,counts,norm,rot", APPENDS)
def test_append_and_read(heads, kv, dim, page, starts, counts, norm, rot):
    rng = np.random.default_rng(heads * 1000 + dim)
    pool = Pool(rng, heads, kv, dim, page, counts)
    n = sum(counts)
    q, k, v = rows_of(rng, n, heads, dim), rows_of(rng, n, kv, dim), rows_of(rng, n, kv, dim)
    wq, wk = (rng.standard_normal(dim).astype(np.float32) if norm else None for _ in range(2))
    cos, sin = R.rope(max(counts), dim) if rot else (None, None)
    got = pool.append(starts, counts, q, k, v, q_norm=wq, k_norm=wk, eps=EPS, cos=cos, sin=sin)
    pos = np.concatenate([np.arange(a, a + c) for a, c in zip(starts, counts)])
    at = (lambda t: t[pos][:, None]) if rot else (lambda t: None)
    once(got, R.turn(q, wq, EPS, at(cos), at(sin)))
    k64 = R.turn(k, wk, EPS, at(cos), at(sin)).astype(np.float32)
    want_k = np.concatenate([R.quantize(x) for x in np.split(k64, np.cumsum(counts)[:-1])])
    want_v = np.concatenate([R.quantize(x) for x in np.split(v, np.cumsum(counts)[:-1])])
    got_k, got_v = pool.read(starts, counts)
    assert np.array_equal(got_k, want_k.astype(np.float32)) and np.array_equal(got_v, want_v.astype(np.float32))


@pytest.mark.parametrize("dim,page,pieces", [
    (64, 16, [1] * 40),
    (64, 64, [5, 11, 1, 16, 15, 17, 33, 2]),
    (128, 32, [7, 64, 30, 1, 1, 50]),
    (32, 48, [20, 40, 13]),
    (256, 16, [3, 31, 14, 40]),
])
def test_append_in_pieces_is_append_at_once(dim, page, pieces):
    """Codes depend on the values alone: after every piece the cache is the
    quantization of the fp32 rows so far, also where a piece spans blocks
    whose parity the open-block store has to hand over."""
    rng = np.random.default_rng(dim + len(pieces))
    kv, total = 2, sum(pieces)
    pool = Pool(rng, 4, kv, dim, page, [total, total])
    k, v = rows_of(rng, 2 * total, kv, dim).reshape(2, total, kv, dim), rows_of(rng, 2 * total, kv, dim).reshape(2, total, kv, dim)
    at = 0
    for n in pieces:
        two = lambda x: np.concatenate([x[0, at:at + n], x[1, at:at + n]])  # noqa: E731
        pool.append([at, at], [n, n], None, two(k), two(v))
        at += n
        gk, gv = pool.read([0, 0], [at, at])
        for i in range(2):
            assert np.array_equal(gk[i * at:(i + 1) * at], R.quantize(k[i, :at]).astype(np.float32))
            assert np.array_equal(gv[i * at:(i + 1) * at], R.quantize(v[i, :at]).astype(np.float32))


def test_append_taken_back():
    """A sequence goes back into the block before its last one and on."""
    rng = np.random.default_rng(5)
    pool = Pool(rng, 2, 1, 64, 32, [100])
    k, v = rows_of(rng, 100, 1, 64), rows_of(rng, 100, 1, 64)
    pool.append([0], [60], None, k[:60], v[:60])
    for back in (58, 49, 37, 33, 32):  # 60 rows: the block before the last starts at 32
        new_k, new_v = rows_of(rng, 60 - back, 1, 64), rows_of(rng, 60 - back, 1, 64)
        k[back:60], v[back:60] = new_k, new_v
        pool.append([back], [60 - back], None, new_k, new_v)
        gk, gv = pool.read([0], [60])
        assert np.array_equal(gk, R.quantize(k[:60]).astype(np.float32))
        assert np.array_equal(gv, R.quantize(v[:60]).astype(np.float32))


def test_append_quantizer_borders():
    """Ties, zeros, tiny and huge values, and blocks with inf or NaN."""
    rng = np.random.default_rng(6)
    dim, n = 64, 16 * 8
    pool = Pool(rng, 1, 1, dim, 16, [n])
    k = rows_of(rng, n, 1, dim)
    k[0:16] = 0
    k[16:32] = rng.integers(-254, 255, (16, 1, dim)) * 0.5  # scale 1: every odd multiple of a half is a tie
    k[16, 0, 0] = 127.0
    k[32:48] = np.float32(1e-45) * rng.integers(-3, 4, (16, 1, dim))
    k[48:64] *= np.float32(1e37)
    k[64:80] *= np.float32(1e-38)
    k[85, 0, 3] = np.inf
    k[100, 0, 7] = np.nan
    v = np.ascontiguousarray(k[::-1])
    pool.append([0], [n], None, k, v)
    gk, gv = pool.read([0], [n])
    with np.errstate(over="ignore"):
        for got, rows in ((gk, k), (gv, v)):
            want = R.quantize(rows).astype(np.float32)
            assert np.array_equal(got, want, equal_nan=True)
    assert np.isnan(gk[80:112]).all() and np.isfinite(gk[:80]).all() and np.isfinite(gk[112:]).all()


def test_append_strided_in_place_and_rows_behind():
    """q, k, v inside one fused row, q rotated in place; the floats between
    the rows and behind the last one, and pages of nobody, stay."""
    rng = np.random.default_rng(7)
    heads, kv, dim, n = 4, 2, 64, 21
    pool = Pool(rng, heads, kv, dim, 32, [n])
    row = (heads + 2 * kv) * dim + 5
    fused = rng.standard_normal((n + 2, row)).astype(np.float32)
    cos, sin = R.rope(n, dim)
    fb, cb, sb = (H.DeviceBuffer.from_array(a) for a in (fused, cos, sin))
    before = [b.download(np.uint8) for b in pool.bufs[:3]]
    p = pool.plan([0], [n])
    at = lambda off: fb.ptr + 4 * off  # noqa: E731
    p.append(pool.layer, at(1), at(1 + heads * dim), at(1 + (heads + kv) * dim), at(1), q_stride=row, k_stride=row, v_stride=row,
             q_out_stride=row, cos=cb.ptr, sin=sb.ptr, positions=n)
    H.synchronize()
    after = fb.download(np.float32).reshape(fused.shape)
    q = fused[:n, 1:1 + heads * dim].reshape(n, heads, dim)
    once(after[:n, 1:1 + heads * dim].reshape(n, heads, dim), R.turn(q, None, 0, cos[:, None], sin[:, None]))
    after[:n, 1:1 + heads * dim] = fused[:n, 1:1 + heads * dim]
    assert np.array_equal(after, fused)
    gk, _ = pool.read([0], [n])
    k = fused[:n, 1 + heads * dim:1 + (heads + kv) * dim].reshape(n, kv, dim)
    assert np.array_equal(gk, R.quantize(R.turn(k, None, 0, cos[:, None], sin[:, None]).astype(np.float32)).astype(np.float32))
    mine = pool.tables[0, :1]
    for b, old in zip(pool.bufs[:3], before):
        old, new = old.reshape(pool.shape.pages, -1), b.download(np.uint8).reshape(pool.shape.pages, -1)
        others = [i for i in range(pool.shape.pages) if i not in mine]
        assert np.array_equal(old[others], new[others])


ATTENTION = [
    # heads, kv, dim, page, starts, counts
    (4, 2, 64, 16, [0], [1]),                          # one position
    (9, 3, 64, 64, [299], [1]),
    (14, 2, 64, 32, [15, 16, 17, 63, 64, 65, 0], [1] * 7),  # block and tile borders
    (4, 4, 32, 16, [100, 0, 40], [1, 0, 1]),           # a sequence without tokens
    (24, 3, 96, 48, [500, 33], [1, 1]),
    (8, 1, 256, 128, [257, 3], [1, 2]),
    (16, 1, 128, 16, [130], [1]),                      # 16 heads of one key head
    (40, 1, 64, 16, [70], [1]),                        # more than 16
    (5, 1, 160, 32, [90, 7], [1, 3]),
    (14, 2, 64, 64, [5000], [1]),                      # a long history
    (2, 2, 128, 256, [9000, 20, 700], [1, 1, 1]),      # ragged, one much longer
    (32, 8, 128, 16, [40, 100, 3], [4, 3, 5]),         # drafts
    (9, 3, 64, 64, [1000], [7]),
    (14, 2, 64, 64, [0], [70]),                        # prompts
    (9, 3, 64, 32, [0, 0, 0], [33, 130, 17]),
    (4, 2, 128, 64, [100, 17], [150, 65]),             # chunks
    (3, 1, 96, 16, [31], [100]),
    (2, 1, 256, 32, [5], [90]),
    (6, 2, 32, 16, [0], [200]),
    (20, 2, 64, 64, [3000], [40]),                     # a short chunk over a long history
    (8, 2, 64, 32, [300, 0, 77, 12], [1, 90, 5, 1]),   # all kinds together
    (1, 1, 64, 16, [0], [300]),
]


@pytest.mark.parametrize("heads,kv,dim,page,starts,counts", ATTENTION)
def test_attention(heads, kv, dim, page, starts, counts):
    rng = np.random.default_rng(heads * 7919 + dim + sum(starts))
    lens = [a + c for a, c in zip(starts, counts)]
    pool = Pool(rng, heads, kv, dim, page, lens)
    k = [rows_of(rng, n, kv, dim, 0.3) for n in lens]
    v = [rows_of(rng, n, kv, dim, 0.5) for n in lens]
    pool.append([0] * len(lens), lens, None, np.concatenate(k), np.concatenate(v))
    q = rows_of(rng, sum(counts), heads, dim, 0.5)
    scale = 1.0 / np.sqrt(dim)
    got = pool.attention(starts, counts, q, scale)
    at = 0
    for i, (a, c) in enumerate(zip(starts, counts)):
        if c:
            kq, vq, qi = R.quantize(k[i]), R.quantize(v[i]), q[at:at + c]
            want = R.attend(qi, kq, vq, a, scale)
            off = np.abs(got[at:at + c] - want)
            assert np.isfinite(got[at:at + c]).all()
            assert off.max() <= R.attend_bound(qi, kq, vq, scale), (i, off.max(), R.attend_bound(qi, kq, vq, scale))
        at += c


@pytest.mark.parametrize("starts,counts", [([200], [1]), ([100], [120])])
def test_attention_extremes(starts, counts):
    """Scores of a thousand apart, zero q, values whose blocks differ by 2^40,
    large q: the softmax stays finite and near the 64-bit one."""
    rng = np.random.default_rng(11)
    heads, kv, dim, n = 4, 2, 64, starts[0] + counts[0]
    pool = Pool(rng, heads, kv, dim, 32, [n])
    k, v = rows_of(rng, n, kv, dim, 0.0), rows_of(rng, n, kv, dim, 0.0)
    k[37] *= 100
    v[48:64] *= np.float32(2.0**20)
    v[80:96] *= np.float32(2.0**-20)
    pool.append([0], [n], None, k, v)
    q = rows_of(rng, counts[0], heads, dim, 0.0)
    q[:, 0] = 0
    q[:, 1] *= 50
    q[:, 2] *= np.float32(2.0**-30)
    got = pool.attention(starts, counts, q, 0.125)
    kq, vq = R.quantize(k), R.quantize(v)
    want = R.attend(q, kq, vq, starts[0], 0.125)
    for h in range(heads):
        bound = R.attend_bound(q[:, h:h + 1], kq[:, h // 2:h // 2 + 1], vq[:, h // 2:h // 2 + 1], 0.125)
        assert np.abs(got[:, h] - want[:, h]).max() <= bound


@pytest.mark.parametrize("count", [1, 40])
def test_attention_sees_only_what_it_may(count):
    """A block with NaN is seen by the rows that attend a position of it and by
    no other; everything behind the batch's last position is NaN already
    (Pool) and never seen."""
    rng = np.random.default_rng(12)
    n, dim = 64 + count, 64
    pool = Pool(rng, 2, 1, dim, 32, [n])
    k, v = rows_of(rng, n, 1, dim, 0.0), rows_of(rng, n, 1, dim, 0.0)
    bad_k, bad_v = k.copy(), v.copy()
    bad_k[64:64 + count, 0] = k[64:64 + count, 0]
    first = 64 + (17 if count > 17 else 0)  # in the second new block
    bad_v[first, 0, 5] = np.nan
    bad_k[min(first + 16, n - 1), 0, 9] = np.inf
    q = rows_of(rng, count, 2, dim, 0.0)
    pool.append([0], [n], None, bad_k, bad_v)
    got = pool.attention([64], [count], q, 0.125)
    want = R.attend(q, R.quantize(bad_k), R.quantize(bad_v), 64, 0.125)
    assert np.array_equal(np.isnan(got), np.isnan(want))
    ok = ~np.isnan(want)
    if ok.any():
        assert np.abs(got[ok] - want[ok]).max() <= R.attend_bound(q, R.quantize(k), R.quantize(v), 0.125)


def test_attention_strided_and_rows_behind():
    rng = np.random.default_rng(13)
    heads, kv, dim, n = 6, 2, 64, 50
    pool = Pool(rng, heads, kv, dim, 32, [n])
    k, v = rows_of(rng, n, kv, dim), rows_of(rng, n, kv, dim)
    pool.append([0], [n], None, k, v)
    for count in (1, 30):
        q = rng.standard_normal((count + 1, heads * dim + 3)).astype(np.float32)
        out = np.full((count + 1, heads * dim + 7), 7.0, np.float32)
        qb, ob = H.DeviceBuffer.from_array(q), H.DeviceBuffer.from_array(out)
        p = pool.plan([n - count], [count])
        p.attention(pool.layer, qb.ptr + 4, 0.125, ob.ptr + 8, q_stride=heads * dim + 3, out_stride=heads * dim + 7)
        H.synchronize()
        got = ob.download(np.float32).reshape(out.shape)
        qq = q[:count, 1:1 + heads * dim].reshape(count, heads, dim)
        want = R.attend(qq, R.quantize(k), R.quantize(v), n - count, 0.125)
        mine = got[:count, 2:2 + heads * dim].reshape(count, heads, dim).copy()
        assert np.abs(mine - want).max() <= R.attend_bound(qq, R.quantize(k), R.quantize(v), 0.125)
        got[:count, 2:2 + heads * dim] = 7.0
        assert (got == 7.0).all()
        # In place.
        p.attention(pool.layer, qb.ptr + 4, 0.125, qb.ptr + 4, q_stride=heads * dim + 3, out_stride=heads * dim + 3)
        H.synchronize()
        again = qb.download(np.float32).reshape(q.shape)[:count, 1:1 + heads * dim].reshape(count, heads, dim)
        assert np.array_equal(again, mine)


def test_shared_prefix_pages():
    """Two sequences read the same full pages and write their own; forks of a
    prompt without a copy."""
    rng = np.random.default_rng(14)
    heads, kv, dim, page = 4, 2, 64, 32
    pool = Pool(rng, heads, kv, dim, page, [64, 100, 90])
    prefix_k, prefix_v = rows_of(rng, 64, kv, dim), rows_of(rng, 64, kv, dim)
    pool.append([0], [64], None, prefix_k, prefix_v, rows=[0])
    for i in (1, 2):
        pool.tables[i, :2] = pool.tables[0, :2]
    ends = [36, 26]
    k, v = [rows_of(rng, n, kv, dim) for n in ends], [rows_of(rng, n, kv, dim) for n in ends]
    pool.append([64, 64], ends, None, np.concatenate(k), np.concatenate(v), rows=[1, 2])
    q = rows_of(rng, 2, heads, dim)
    got = pool.attention([99, 89], [1, 1], q, 0.125, rows=[1, 2])
    for i in range(2):
        kk, vv = R.quantize(np.concatenate([prefix_k, k[i]])), R.quantize(np.concatenate([prefix_v, v[i]]))
        want = R.attend(q[i:i + 1], kk, vv, len(kk) - 1, 0.125)
        assert np.abs(got[i] - want[0]).max() <= R.attend_bound(q[i:i + 1], kk, vv, 0.125)


def test_decode_steps_replayed_from_a_graph():
    """append + attention of one token per sequence captured once and replayed
    step after step, the batch set between the replays (lengths, block borders
    and, at the end, one sequence fewer), against the eager calls."""
    rng = np.random.default_rng(15)
    heads, kv, dim, page, n0 = 6, 2, 64, 32, [5, 30, 200]
    steps = 24
    pools = [Pool(np.random.default_rng(16), heads, kv, dim, page, [n + steps for n in n0]) for _ in range(2)]
    k0, v0 = rows_of(rng, sum(n0), kv, dim), rows_of(rng, sum(n0), kv, dim)
    for pool in pools:
        pool.append([0, 0, 0], n0, None, k0, v0)
    cos, sin = R.rope(400, dim)
    cb, sb = H.DeviceBuffer.from_array(cos), H.DeviceBuffer.from_array(sin)
    bufs = [[H.DeviceBuffer.from_array(np.zeros(3 * h * dim, np.float32)) for h in (heads, kv, kv, heads, heads)] for _ in pools]
    plans = [H.Kv8Plan(pool.shape, 3, 3, pool.tables.size) for pool in pools]

    def step(i):
        q, k, v, qo, o = (b.ptr for b in bufs[i])
        plans[i].append(pools[i].layer, q, k, v, qo, cos=cb.ptr, sin=sb.ptr, positions=400)
        plans[i].attention(pools[i].layer, qo, 0.125, o)

    for p, pool in zip(plans, pools):
        p.set(pool.slots, n0, [1, 1, 1], pool.tables)
    H.synchronize()
    graph = H.Graph(lambda: step(0))
    with pytest.raises(H.HipError, match="rotation tables"):
        plans[0].set(pools[0].slots[:1], [400], [1], np.arange(13)[None])
    for n in range(steps):
        counts = [1, 1, 1] if n < steps - 2 else [1, 0, 1]
        new = [rows_of(rng, 3, h, dim) for h in (heads, kv, kv)]
        starts = [a + n for a in n0]
        outs = []
        for i in range(2):
            for b, x in zip(bufs[i], new):
                b.upload(x)
            plans[i].set(pools[i].slots, starts, counts, pools[i].tables)
            if i == 0:
                graph.launch()
            else:
                step(1)
            H.synchronize()
            outs.append(bufs[i][4].download(np.float32).reshape(3, -1)[:sum(counts)])
        assert np.array_equal(outs[0], outs[1]), n
        assert np.isfinite(outs[0]).all()
    for a, b in zip(pools[0].bufs[:2], pools[1].bufs[:2]):
        assert np.array_equal(a.download(np.uint8), b.download(np.uint8))


@pytest.mark.parametrize("empty", [True, False])
def test_every_kind_of_batch_from_one_graph(empty):
    """A graph captured with an empty batch (or with drafts and a prompt)
    replayed for single tokens, drafts, prompts and mixtures, long and short,
    against eager calls; one captured for single tokens refuses a prompt."""
    rng = np.random.default_rng(21)
    heads, kv, dim, page, n = 8, 2, 64, 32, 3
    pool = Pool(rng, heads, kv, dim, page, [2600, 700, 300])
    k, v = rows_of(rng, 3600, kv, dim), rows_of(rng, 3600, kv, dim)
    pool.append([0, 0, 0], [2600, 700, 300], None, k, v)
    plan = H.Kv8Plan(pool.shape, n, 400, pool.tables.size)
    qb, ob = (H.DeviceBuffer(400 * heads * dim * 4) for _ in range(2))
    plan.set(pool.slots, [0] * n, [0, 0, 0] if empty else [4, 60, 0], pool.tables)
    H.synchronize()
    graph = H.Graph(lambda: plan.attention(pool.layer, qb.ptr, 0.125, ob.ptr))
    for starts, counts in (([2599, 699, 299], [1, 1, 1]), ([2590, 0, 0], [3, 0, 4]), ([100, 600, 0], [200, 100, 100]), ([2300, 0, 17], [300, 1, 2]), ([5, 6, 7], [1, 0, 0])):
        q = rows_of(rng, sum(counts), heads, dim)
        want = pool.attention(starts, counts, q, 0.125)
        plan.set(pool.slots, starts, counts, pool.tables)
        for _ in range(2):  # the second replay on the same batch
            qb.upload(q)
            ob.upload(np.full(400 * heads * dim, 5.0, np.float32))
            graph.launch()
            H.synchronize()
            got = ob.download(np.float32).reshape(400, heads, dim)
            assert np.array_equal(got[:len(q)], want) and (got[len(q):] == 5.0).all()
    one = H.Kv8Plan(pool.shape, n, 400, pool.tables.size)
    one.set(pool.slots, [9] * n, [1] * n, pool.tables)
    H.synchronize()
    single = H.Graph(lambda: one.attention(pool.layer, qb.ptr, 0.125, ob.ptr))
    for counts in ([2, 1, 1], [100, 1, 1]):
        with pytest.raises(H.HipError, match="captured for"):
            one.set(pool.slots, [9] * n, counts, pool.tables)
    one.set(pool.slots, [2000, 30, 9], [1, 0, 1], pool.tables)
    single.launch()
    H.synchronize()


def new_stream():
    """A stream of the HIP runtime that the library is linked with."""
    import ctypes as C

    s = C.c_void_p()
    create = H.load().hipStreamCreateWithFlags  # found through the library's own dependencies
    create.argtypes = [C.c_void_p, C.c_uint]
    assert create(C.byref(s), 1) == 0
    return s.value


def wait_for(stream):
    import ctypes as C

    wait = H.load().hipStreamSynchronize
    wait.argtypes = [C.c_void_p]
    assert wait(stream) == 0


def test_two_plans_on_two_streams():
    rng = np.random.default_rng(17)
    heads, kv, dim = 8, 2, 64
    n = [3000, 2500]
    pools = [Pool(rng, heads, kv, dim, 64, [m]) for m in n]
    rows = []
    for pool, m in zip(pools, n):
        k, v = rows_of(rng, m, kv, dim), rows_of(rng, m, kv, dim)
        pool.append([0], [m], None, k, v)
        rows.append((k, v))
    q = [rows_of(rng, 1, heads, dim) for _ in n]
    qb = [H.DeviceBuffer.from_array(x) for x in q]
    ob = [H.DeviceBuffer(x.nbytes) for x in q]
    streams = [new_stream() for _ in n]
    plans = []
    for pool, m, s in zip(pools, n, streams):
        p = H.Kv8Plan(pool.shape, 1, 1, pool.tables.size)
        p.set(pool.slots, [m - 1], [1], pool.tables, stream=s)
        plans.append(p)
    for _ in range(20):
        for i in range(2):
            plans[i].attention(pools[i].layer, qb[i].ptr, 0.125, ob[i].ptr, stream=streams[i])
    for s in streams:
        wait_for(s)
    for i in range(2):
        kk, vv = R.quantize(rows[i][0]), R.quantize(rows[i][1])
        want = R.attend(q[i], kk, vv, n[i] - 1, 0.125)
        assert np.abs(ob[i].download(np.float32).reshape(want.shape) - want).max() <= R.attend_bound(q[i], kk, vv, 0.125)


def test_pool_past_four_gigabytes():
    """Pages at the end of a pool of more than 2^32 bytes of keys."""
    rng = np.random.default_rng(18)
    heads, kv, dim, page, n = 4, 2, 128, 256, 600
    pages = (1 << 32) // (kv * dim * page) + 40
    shape = H.Kv8Shape(heads, kv, dim, page, pages, 1)
    code, scale, opened = shape.sizes()
    assert code > 1 << 32
    bufs = [H.DeviceBuffer(x) for x in (code, code, 4 * scale, 4 * opened)]
    layer = H.Kv8Layer(*(b.ptr for b in bufs))
    table = np.array([[pages - 1, 0, pages - 7]], np.int32)
    k, v, q = rows_of(rng, n, kv, dim), rows_of(rng, n, kv, dim), rows_of(rng, n, heads, dim)
    p = H.Kv8Plan(shape, 1, n)
    p.set([0], [0], [n], table)
    kb, vb, qb = (H.DeviceBuffer.from_array(x) for x in (k, v, q))
    ob = H.DeviceBuffer(q.nbytes)
    p.append(layer, None, kb.ptr, vb.ptr, None)
    p.attention(layer, qb.ptr, 0.1, ob.ptr)
    gk = H.DeviceBuffer(k.nbytes)
    p.read(layer, gk.ptr, None)
    H.synchronize()
    assert np.array_equal(gk.download(np.float32).reshape(k.shape), R.quantize(k).astype(np.float32))
    got = ob.download(np.float32).reshape(q.shape)
    p.set([0], [n - 1], [1], table)
    p.attention(layer, qb.ptr + 4 * (n - 1) * heads * dim, 0.1, ob.ptr)
    H.synchronize()
    one = ob.download(np.float32).reshape(q.shape)[0]
    kk, vv = R.quantize(k), R.quantize(v)
    want = R.attend(q, kk, vv, 0, 0.1)
    bound = R.attend_bound(q, kk, vv, 0.1)
    assert np.abs(got - want).max() <= bound and np.abs(one - want[-1]).max() <= bound


def test_nothing_to_do():
    rng = np.random.default_rng(19)
    pool = Pool(rng, 2, 1, 64, 16, [10])
    before = [b.download(np.uint8) for b in pool.bufs]
    for starts, counts, rows in (([], [], []), ([4], [0], [0])):
        p = pool.plan(starts, counts, rows=rows)
        one = H.DeviceBuffer.from_array(np.full(128, 3.0, np.float32))
        p.append(pool.layer, one.ptr, one.ptr, one.ptr, one.ptr)
        p.attention(pool.layer, one.ptr, 1.0, one.ptr)
        p.read(pool.layer, one.ptr, one.ptr)
        H.synchronize()
        assert (one.download(np.float32) == 3.0).all()
    assert all(np.array_equal(a, b.download(np.uint8)) for a, b in zip(before, pool.bufs))


def test_refusals():
    rng = np.random.default_rng(20)
    pool = Pool(rng, 2, 1, 64, 16, [40, 40])
    b = H.DeviceBuffer(1 << 16)
    no = lambda match: pytest.raises(H.HipError, match=match)  # noqa: E731
    fresh = H.Kv8Plan(pool.shape, 2, 64)
    with no("no batch set"):
        fresh.append(pool.layer, b.ptr, b.ptr, b.ptr, b.ptr)
    with no("no batch set"):
        fresh.attention(pool.layer, b.ptr, 1.0, b.ptr)
    with no("no batch set"):
        fresh.read(pool.layer, b.ptr, b.ptr)
    with no("more tokens"):
        fresh.set([0], [0], [65], np.arange(5)[None])
    with no("more sequences"):
        fresh.set([0, 1, 1], [0, 0, 0], [1, 1, 1], np.arange(3)[:, None])
    with no("no batch set"):  # a refused batch leaves none behind
        fresh.read(pool.layer, b.ptr, b.ptr)
    p = pool.plan([0, 0], [20, 20])
    for kw, match in ((dict(q_stride=127), "shorter"), (dict(k_stride=63), "shorter"), (dict(v_stride=63), "shorter"),
                      (dict(q_out_stride=100), "shorter"), (dict(q_norm=b.ptr), "go together"), (dict(cos=b.ptr), "go together"),
                      (dict(cos=b.ptr, sin=b.ptr, positions=19), "fewer positions"),
                      (dict(q_norm=b.ptr, k_norm=b.ptr, eps=-1.0), "eps"), (dict(q_stride=200), "equal strides")):
        with no(match):
            p.append(pool.layer, b.ptr, b.ptr, b.ptr, b.ptr, **kw)
    with no("null"):
        p.append(pool.layer, b.ptr, None, b.ptr, b.ptr)
    with no("q_out"):
        p.append(pool.layer, b.ptr, b.ptr, b.ptr, None)
    with no("null"):
        p.attention(pool.layer, None, 1.0, b.ptr)
    with no("finite"):
        p.attention(pool.layer, b.ptr, float("nan"), b.ptr)
    with no("shorter"):
        p.attention(pool.layer, b.ptr, 1.0, b.ptr, out_stride=1)
    with no("shorter"):
        p.read(pool.layer, b.ptr, b.ptr, v_stride=1)
    bad = H.Kv8Layer(pool.layer.k + 4, pool.layer.v, pool.layer.scales, pool.layer.open)
    with no("aligned"):
        p.read(bad, b.ptr, b.ptr)
    with no("null"):
        p.read(H.Kv8Layer(None, pool.layer.v, pool.layer.scales, pool.layer.open), b.ptr, b.ptr)
    # Batches that are read but not appended to.
    shared = pool.tables.copy()
    shared[1] = shared[0]
    r = H.Kv8Plan(pool.shape, 2, 64, 16)
    for slots, tables, match in ((pool.slots, shared, "twice"), (np.array([1, 1]), pool.tables, "same slot"),
                                 (None, pool.tables, "without slots")):
        r.set(slots, [0, 0], [20, 20], tables)
        with no(match):
            r.append(pool.layer, None, b.ptr, b.ptr, None)
        r.read(pool.layer, b.ptr, None)
    H.synchronize()


def test_rows_past_32_bits_refused():
    with pytest.raises(H.HipError, match="2\\^30 rows"):
        H.Kv8Plan(H.Kv8Shape(4096, 1, 32, 16, 4, 1), 1, (1 << 18) + 1)


LONG = [
    # heads, kv, dim, page, starts, counts: single tokens and drafts whose histories are taken in pieces
    (9, 3, 64, 64, [5200, 40], [1, 1]),
    (5, 1, 32, 16, [4100], [1]),
    (8, 2, 128, 32, [4000, 3500], [4, 1]),
    (40, 1, 64, 16, [3600], [1]),
    (16, 2, 96, 48, [3300], [2]),
    (7, 1, 160, 64, [2500], [3]),
    (8, 1, 256, 128, [2700, 2000], [1, 2]),
]


@pytest.mark.parametrize("heads,kv,dim,page,starts,counts", LONG)
def test_attention_in_pieces_eager_and_replayed(heads, kv, dim, page, starts, counts):
    """Long histories, against the formula, and the same bits from a graph
    that is replayed between batches of other lengths."""
    rng = np.random.default_rng(heads * 131 + dim)
    lens = [a + c for a, c in zip(starts, counts)]
    pool = Pool(rng, heads, kv, dim, page, lens)
    k, v = ([rows_of(rng, n, kv, dim, s) for n in lens] for s in (0.3, 0.5))
    pool.append([0] * len(lens), lens, None, np.concatenate(k), np.concatenate(v))
    scale = 1.0 / np.sqrt(dim)
    plan = H.Kv8Plan(pool.shape, len(lens), sum(counts), pool.tables.size)
    qb, ob = (H.DeviceBuffer(sum(counts) * heads * dim * 4) for _ in range(2))
    plan.set(pool.slots, [3] * len(lens), counts, pool.tables)
    H.synchronize()
    graph = H.Graph(lambda: plan.attention(pool.layer, qb.ptr, scale, ob.ptr))
    for at in (starts, [min(100, s) for s in starts], starts):
        q = rows_of(rng, sum(counts), heads, dim, 0.5)
        got = pool.attention(at, counts, q, scale)
        plan.set(pool.slots, at, counts, pool.tables)
        qb.upload(q)
        graph.launch()
        H.synchronize()
        assert np.array_equal(ob.download(np.float32).reshape(q.shape), got)
        row = 0
        for i, c in enumerate(counts):
            kq, vq, qi = R.quantize(k[i])[:at[i] + c], R.quantize(v[i])[:at[i] + c], q[row:row + c]
            off = np.abs(got[row:row + c] - R.attend(qi, kq, vq, at[i], scale)).max()
            assert off <= R.attend_bound(qi, kq, vq, scale), (i, off)
            row += c


def test_replayed_batches_larger_than_a_captured_grid():
    """A captured launch has a bounded grid, whose workgroups take further
    units in turn: thousands of sequences, as prompts and as single tokens,
    give the bits of eager calls."""
    heads, dim, page = 8, 32, 16
    prompts, singles, length = 520, 2200, 66
    tokens = prompts * length
    pools = [Pool(np.random.default_rng(33), heads, heads, dim, page, [length + 1] * singles) for _ in range(2)]
    plans = [H.Kv8Plan(pool.shape, singles, tokens, pool.tables.size) for pool in pools]
    n = tokens * heads * dim
    bufs = [[H.DeviceBuffer(n * 4) for _ in range(6)] for _ in pools]

    def step(i):
        q, k, v, o, rk, rv = (b.ptr for b in bufs[i])
        plans[i].append(pools[i].layer, q, k, v, q)
        plans[i].attention(pools[i].layer, q, 0.2, o)
        plans[i].read(pools[i].layer, rk, rv)

    plans[0].set([], [], [], np.zeros((0, 0), np.int32))
    H.synchronize()
    graph = H.Graph(lambda: step(0))
    rng = np.random.default_rng(34)
    for seqs, start, count in ((prompts, 0, length), (singles, 0, 1), (singles, 1, 2), (prompts, 3, 1)):
        rows = [rows_of(rng, seqs * count, heads, dim) for _ in range(3)]
        outs = []
        for i in range(2):
            for b, x in zip(bufs[i], rows):
                b.upload(x)
            plans[i].set(pools[i].slots[:seqs], [start] * seqs, [count] * seqs, pools[i].tables[:seqs])
            if i == 0:
                graph.launch()
            else:
                step(1)
            H.synchronize()
            outs.append([b.download(np.float32)[:seqs * count * heads * dim] for b in bufs[i][3:]])
        for a, b in zip(*outs):
            assert np.isfinite(a).all() and np.array_equal(a, b)


@pytest.mark.parametrize("dim", [64, 256])
@pytest.mark.parametrize("count", [6, 60])
@pytest.mark.parametrize("big", [2.0**20, 2.0**60])
def test_attention_next_to_large_values(count, big, dim):
    """Values far larger than the rest, behind a row's position or under
    scores that leave them no weight, cost the other values no bits: a row's
    error counts against the values that it takes."""
    rng = np.random.default_rng(35)
    start, heads, kv = 61, 4, 2
    n = start + count
    k, v = rows_of(rng, n, kv, dim, 0.0), rows_of(rng, n, kv, dim, 0.0)
    q = rows_of(rng, count, heads, dim, 0.0)
    k[16:32], q[:, :, 0] = 0.0, 4.0
    k[16:32, :, 0] = -160.0  # scores of -80: weights under 2^-100
    v[16:32] *= np.float32(big)
    last = n - 1 - (n - 1) % 16  # the last block: rows before it do not see it
    v[last:] *= np.float32(big)
    pool = Pool(rng, heads, kv, dim, 32, [n])
    pool.append([0], [n], None, k, v)
    got = pool.attention([start], [count], q, 0.125)
    kq, vq = R.quantize(k), R.quantize(v)
    rows = last - start
    assert rows > 0
    want = R.attend(q[:rows], kq[:last], vq[:last], start, 0.125)
    small = vq[:last].copy()
    small[16:32] = 0.0
    bound = R.attend_bound(q[:rows], kq[:last], small, 0.125)
    assert np.abs(want).max() > 20 * bound
    assert np.abs(got[:rows] - want).max() <= bound


@pytest.mark.parametrize("scale", [0.0, -0.2, 0.2])
@pytest.mark.parametrize("count", [1, 6, 70])
def test_attention_odd_rows_and_scales(count, scale):
    """A scale of 0 (the values' mean) and a negative one; a row of q with inf
    or NaN gives NaN and leaves the others alone; blocks of zeros and of
    denormal numbers among the history."""
    rng = np.random.default_rng(36)
    start, heads, kv, dim = 90, 4, 2, 64
    n = start + count
    k, v = rows_of(rng, n, kv, dim, 0.0), rows_of(rng, n, kv, dim, 0.0)
    k[0:16], v[16:32] = 0.0, 0.0
    k[32:48] *= np.float32(1e-40)
    v[48:64] *= np.float32(1e-40)
    pool = Pool(rng, heads, kv, dim, 32, [n])
    pool.append([0], [n], None, k, v)
    q = rows_of(rng, count, heads, dim, 0.0)
    kq, vq = R.quantize(k), R.quantize(v)
    want, bound = R.attend(q, kq, vq, start, scale), R.attend_bound(q, kq, vq, scale)
    q[0, 1, 7], q[count - 1, 2, 63] = np.nan, np.inf
    got = pool.attention([start], [count], q, scale)
    odd = np.zeros((count, heads), bool)
    odd[0, 1] = odd[count - 1, 2] = True
    assert np.isnan(got[odd]).all()
    assert np.abs(got[~odd] - want[~odd]).max() <= bound
