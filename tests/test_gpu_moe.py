"""A layer of experts on the GPU (llmi_hip_moe_*): router, grouped products
and expert MLPs against tests/moe_reference.py, alone and together."""

import ctypes as C

import numpy as np
import pytest

import llmi_hip as H
import moe_reference as R

pytestmark = pytest.mark.gpu

NAN, INF = np.float32("nan"), np.float32("inf")
GUARD = np.float32(-12345.5)


def dev(a):
    return H.DeviceBuffer.from_array(np.ascontiguousarray(a))


class Workspace:
    """A workspace of just the bytes asked for, full of NaNs, with a guard behind it."""

    def __init__(self, nbytes):
        self.n = nbytes
        self.buf = dev(np.full(nbytes // 4 + 64, NAN, np.float32))

    def intact(self):
        assert np.isnan(self.buf.download(np.float32)[self.n // 4:]).all()


def make(rng, qtype, count, out, n_in, spread=1.0):
    data, scales, values = R.matrices(rng, qtype, count, out, n_in, spread)
    d, s = dev(data), dev(scales)
    return H.Experts.upload_dev(d.ptr, s.ptr, count, out, n_in, qtype), values


def pitched(rows, stride):
    """Rows a stride apart, guard values between them."""
    buf = np.full((len(rows), stride), GUARD, np.float32)
    buf[:, :rows.shape[1]] = rows
    return buf


# ------------------------------------------------------------------ router


def run_route(logits, top_k, renormalise=True, scale=1.0, stride=None):
    tokens, experts = logits.shape
    stride = stride or experts
    lb = dev(pitched(logits.astype(np.float32), stride))
    ids, w = dev(np.full((tokens + 1, top_k), 77, np.int32)), dev(np.full((tokens + 1, top_k), GUARD, np.float32))
    H.moe_route(lb.ptr, tokens, experts, top_k, ids.ptr, w.ptr, stride=stride, renormalise=renormalise, scale=scale)
    H.synchronize()
    ids, w = ids.download(np.int32).reshape(-1, top_k), w.download(np.float32).reshape(-1, top_k)
    assert (ids[tokens] == 77).all() and (w[tokens] == GUARD).all()
    return ids[:tokens], w[:tokens]


def check_route(logits, top_k, renormalise=True, scale=1.0, stride=None):
    ids, w = run_route(logits, top_k, renormalise, scale, stride)
    want_ids, want = R.route(logits.astype(np.float32), top_k, renormalise, scale)
    assert np.array_equal(ids, want_ids)
    # exp of a rounded difference (2^-24 of at most 104, below which it is 0) and
    # of two roundings, a sum of up to 16 + 6 additions or of top_k, a quotient, a product.
    span = min(2 * np.abs(np.where(np.isfinite(logits), logits, 0.0)).max(initial=0.0), 104.0)
    assert np.all(np.abs(w - want) <= np.abs(want) * 2.0**-24 * (2 * span + 40 + top_k) + 1e-37 * abs(scale))


@pytest.mark.parametrize("tokens,experts,top_k", [(1, 1, 1), (1, 64, 8), (3, 2, 2), (5, 65, 64), (64, 8, 2), (7, 128, 6),
                                                  (9, 129, 4), (130, 256, 8), (2, 257, 3), (4, 1024, 64), (0, 8, 2)])
@pytest.mark.parametrize("renormalise", [True, False])
def test_route(tokens, experts, top_k, renormalise):
    rng = np.random.default_rng(tokens * 7 + experts)
    check_route(rng.standard_normal((tokens, experts)) * 3, top_k, renormalise, 2.5, experts + 3)


def test_route_ties_and_masks():
    rng = np.random.default_rng(3)
    l = rng.integers(-3, 4, (200, 40)).astype(np.float32)
    l[l == 0] *= np.where(rng.random((l == 0).sum()) < 0.5, -1, 1)  # +0 and -0
    l[rng.random(l.shape) < 0.3] = -INF
    l[rng.random(l.shape) < 0.05] = NAN
    l[0], l[1] = -INF, NAN
    l[2, 1:] = -INF
    l[3] = np.finfo(np.float32).min
    l[4, 7] = l[4, 30] = INF
    l[5, 7] = np.finfo(np.float32).max
    l[6, :] = -INF
    l[6, 39] = np.finfo(np.float32).min
    for renormalise in (True, False):
        check_route(l, 5, renormalise)
        check_route(l, 40, renormalise, -0.5)


# ---------------------------------------------------------- grouped products


def draw_ids(rng, tokens, top_k, count, pad=0.0, skew=1.0):
    p = rng.standard_normal((tokens, count)) + skew * rng.standard_normal(count)
    ids = np.argsort(-p, 1)[:, :top_k].astype(np.int32)
    ids[rng.random(ids.shape) < pad] = -1
    return ids


def run_matmul(experts, ids, x, per_row, x_stride=None, y_stride=None, y0=None, stream=None):
    slots = ids.size
    x_stride, y_stride = x_stride or experts.n_in, y_stride or experts.out
    xb, ib = dev(pitched(x, x_stride)), dev(ids.astype(np.int32).reshape(-1))
    yb = dev(np.full((slots + 1, y_stride), GUARD, np.float32))
    work = Workspace(H.moe_matmul_bytes(experts, slots, per_row))
    H.moe_matmul(experts, ib.ptr, slots, xb.ptr, yb.ptr, work.buf.ptr, work.n, per_row=per_row, x_stride=x_stride, y_stride=y_stride,
                 stream=stream)
    H.synchronize()
    work.intact()
    y = yb.download(np.float32).reshape(slots + 1, y_stride)
    assert (y[slots] == GUARD).all() and (y[:, experts.out:] == GUARD).all()
    return y[:slots, :experts.out]


def some(n, rng):
    """All of n rows, or enough of many."""
    return range(n) if n <= 400 else np.unique(np.concatenate([np.arange(8), n - 1 - np.arange(8), rng.integers(0, n, 150)]))


def check_matmul(y, ids, x, per_row, values):
    flat = ids.reshape(-1)
    assert np.array_equal((y == GUARD).all(1), (flat < 0) | (flat >= len(values)))
    for s in some(len(flat), np.random.default_rng(2)):
        e = flat[s]
        if e < 0 or e >= len(values):
            assert (y[s] == GUARD).all(), s
            continue
        want, bound = R.product(x[int(s) // per_row], values[e])
        assert np.all(np.abs(y[s] - want) <= bound), (s, e, np.abs(y[s] - want).max(), bound.min())


MATMULS = [
    # type, experts, tokens, top_k, in, out, per_row
    (H.Q4_0, 1, 1, 1, 1, 1, 1), (H.Q8_0, 1, 1, 1, 1, 1, 1), (H.Q4_0, 3, 1, 2, 31, 15, 2), (H.Q8_0, 3, 1, 2, 33, 17, 2),
    (H.Q4_0, 8, 1, 2, 576, 96, 2), (H.Q8_0, 8, 1, 8, 127, 64, 8), (H.Q4_0, 5, 7, 3, 129, 65, 3), (H.Q8_0, 5, 7, 3, 100, 130, 1),
    (H.Q4_0, 4, 40, 2, 256, 48, 2), (H.Q8_0, 64, 20, 8, 160, 32, 8), (H.Q4_0, 2, 100, 1, 97, 200, 1), (H.Q8_0, 2, 300, 2, 64, 33, 2),
    (H.Q4_0, 16, 130, 4, 320, 128, 4), (H.Q8_0, 13, 50, 3, 1000, 77, 3), (H.Q4_0, 300, 30, 6, 64, 16, 6),
    # Several rows an expert without a grouping (twice 8 of them), and just too many for that.
    (H.Q4_0, 3, 16, 2, 200, 70, 2), (H.Q8_0, 1, 16, 1, 130, 40, 1), (H.Q8_0, 1, 17, 1, 130, 40, 1), (H.Q4_0, 4, 6, 3, 64, 6000, 3),
    # Long work: more slots than the kernel for short work takes.
    (H.Q4_0, 8, 500, 2, 100, 4112, 2), (H.Q8_0, 8, 900, 1, 192, 4090, 1), (H.Q4_0, 2, 1300, 1, 33, 4100, 1), (H.Q8_0, 70, 1200, 3, 64, 2048, 3),
    # Each way of grouping: by every workgroup (above), by one, by several.
    (H.Q4_0, 8, 1500, 2, 32, 16, 2), (H.Q8_0, 100, 2047, 1, 40, 20, 1), (H.Q8_0, 100, 2049, 1, 40, 20, 1), (H.Q4_0, 40, 4500, 2, 33, 17, 2),
    (H.Q8_0, 4, 5000, 1, 24, 2100, 1), (H.Q4_0, 2000, 2100, 2, 32, 16, 1),
]


@pytest.mark.parametrize("qtype,count,tokens,top_k,n_in,out,per_row", MATMULS)
def test_matmul(qtype, count, tokens, top_k, n_in, out, per_row):
    rng = np.random.default_rng(n_in * 31 + out)
    experts, values = make(rng, qtype, count, out, n_in)
    ids = draw_ids(rng, tokens, top_k, count, 0.1 if tokens > 1 else 0.0)
    x = (rng.standard_normal((-(-ids.size // per_row), n_in)) * np.exp(rng.standard_normal(n_in))).astype(np.float32)
    y = run_matmul(experts, ids, x, per_row, n_in + 5, out + 3)
    check_matmul(y, ids, x, per_row, values)


def test_matmul_ids():
    """Ids of no expert, the same one for all, and some of none."""
    rng = np.random.default_rng(5)
    experts, values = make(rng, H.Q4_0, 6, 40, 96)
    x = rng.standard_normal((150, 96)).astype(np.float32)
    for ids in (np.full(150, -1), np.full(150, 5), np.full(150, 6), np.array([-1, 2**31 - 1, -2**31, 7, 0] * 30), np.arange(150) % 6,
                np.repeat([0, 5], 75)):
        check_matmul(run_matmul(experts, ids.astype(np.int32), x, 1), ids, x, 1, values)
    assert run_matmul(experts, np.zeros(0, np.int32), x[:0], 1).shape == (0, 40)


@pytest.mark.parametrize("qtype", [H.Q4_0, H.Q8_0])
@pytest.mark.parametrize("tokens", [1, 3, 90])
def test_matmul_extremes(qtype, tokens):
    """Rows of very large, very small and zero elements, and of wide spread."""
    rng = np.random.default_rng(11)
    experts, values = make(rng, qtype, 3, 50, 200, 0.3)
    x = rng.standard_normal((tokens, 200))
    x *= np.exp(np.linspace(-85, 80, tokens)[:, None] if tokens > 1 else 60)
    x[0, ::2] *= 1e-30
    x[tokens // 2] *= np.exp(rng.uniform(-40, 0, 200))
    x[-1] = 0 if tokens > 1 else x[-1]
    x = x.astype(np.float32)
    ids = draw_ids(rng, tokens, 1, 3)
    y = run_matmul(experts, ids, x, 1)
    for s, e in enumerate(ids.reshape(-1)):
        want, bound = R.product(x[s], values[e])
        assert np.all(np.abs(y[s] - want) <= bound + 1e-38), s


@pytest.mark.parametrize("qtype", [H.Q4_0, H.Q8_0])
@pytest.mark.parametrize("slots,out", [(3, 40), (150, 40), (1300, 4100)])
@pytest.mark.parametrize("small", [-8, -14, -18, -24, -32])
def test_matmul_small_beside_large(qtype, slots, out, small):
    """Elements 2^small of their row's largest, which a weight of 0 takes out: what is left of them shows."""
    rng = np.random.default_rng(60)
    count, n_in = 3, 100
    data, scales, values = R.matrices(rng, qtype, count, out, n_in)
    data[..., 0] = 0 if qtype == H.Q8_0 else (data[..., 0] & 0xF0) | 8
    values[..., 0] = 0
    d, s = dev(data), dev(scales)
    experts = H.Experts.upload_dev(d.ptr, s.ptr, count, out, n_in, qtype)
    ids = rng.integers(0, count, slots).astype(np.int32)
    x = (rng.standard_normal((slots, n_in)) * 2.0**small).astype(np.float32)
    x[:, 0] = 1.5
    check_matmul(run_matmul(experts, ids, x, 1), ids, x, 1, values)


@pytest.mark.parametrize("tokens", [1, 5, 80])
def test_matmul_nonfinite_rows(tokens):
    """inf and NaN stay in their rows; a row with an inf keeps the signs of the products that decide."""
    rng = np.random.default_rng(12)
    experts, values = make(rng, H.Q8_0, 2, 33, 140)
    x = rng.standard_normal((tokens, 140)).astype(np.float32)
    bad = {0: (17, INF)} if tokens == 1 else {0: (17, INF), 2: (0, -INF), 3: (139, NAN)}
    for t, (i, v) in bad.items():
        x[t, i] = v
    ids = draw_ids(rng, tokens, 1, 2)
    y = run_matmul(experts, ids, x, 1)
    for s, e in enumerate(ids.reshape(-1)):
        if s in bad:
            with np.errstate(invalid="ignore"):
                col = values[e][:, bad[s][0]] * np.float64(bad[s][1])
            assert np.array_equal(np.isnan(y[s]), np.isnan(col)) and np.array_equal(np.sign(y[s])[~np.isnan(col)], np.sign(col)[~np.isnan(col)])
            assert not np.isfinite(y[s]).any()
        else:
            want, bound = R.product(x[s], values[e])
            assert np.all(np.abs(y[s] - want) <= bound)


def test_experts_from_weights():
    """The same experts from planar memory, from weights and from GGUF tensors: the same bits."""
    rng = np.random.default_rng(21)
    for qtype in (H.Q4_0, H.Q8_0):
        n_in, out, count = 75, 37, 3
        data, scales, values = R.matrices(rng, qtype, count, out, n_in)
        d, s = dev(data), dev(scales)
        a = H.Experts.upload_dev(d.ptr, s.ptr, count, out, n_in, qtype)
        b = H.Experts.from_weights([H.Weight.upload(data[e], scales[e], out, n_in, qtype) for e in range(count)])
        ids = np.arange(9, dtype=np.int32) % 4 - 1
        x = rng.standard_normal((9, n_in)).astype(np.float32)
        ya, yb = run_matmul(a, ids, x, 1), run_matmul(b, ids, x, 1)
        assert np.array_equal(ya.view(np.uint32), yb.view(np.uint32))
        check_matmul(ya, ids, x, 1, values)


# ------------------------------------------------------------------- MLPs


class Layer:
    def __init__(self, rng, qtype, down_type, count, hidden, ffn):
        self.gate, self.vg = make(rng, qtype, count, ffn, hidden, 0.3)
        self.up, self.vu = make(rng, qtype, count, ffn, hidden, 0.3)
        self.down, self.vd = make(rng, down_type, count, hidden, ffn, 0.3)

    def run(self, ids, weights, x, residual=None, pad=0, in_place=False, stream=None):
        tokens, top_k = ids.shape
        hidden = self.gate.n_in
        xs, rs, ys = hidden + pad, hidden + 2 * pad, hidden + (2 * pad if in_place else 3 * pad)
        xb, ib, wb = dev(pitched(x, xs)), dev(ids.astype(np.int32)), dev(weights.astype(np.float32))
        rb = None if residual is None else dev(pitched(residual, rs))
        yb = dev(np.full((tokens + 1, ys), GUARD, np.float32))
        if in_place:
            yb = dev(np.concatenate([pitched(residual, rs), np.full((1, rs), GUARD, np.float32)]))
            rb = yb
        work = Workspace(H.moe_mlp_bytes(self.gate, self.down, tokens, top_k))
        H.moe_mlp(self.gate, self.up, self.down, ib.ptr, wb.ptr, tokens, top_k, xb.ptr, yb.ptr, work.buf.ptr, work.n,
                  residual=None if rb is None else rb.ptr, x_stride=xs, residual_stride=rs, y_stride=ys, stream=stream)
        H.synchronize()
        work.intact()
        y = yb.download(np.float32).reshape(tokens + 1, ys)
        assert (y[tokens] == GUARD).all() and (y[:, hidden:] == GUARD).all()
        return y[:tokens, :hidden]

    def check(self, y, ids, weights, x, residual=None):
        top_k = ids.shape[1]
        for t in some(len(ids), np.random.default_rng(3)):
            want, bound, size = np.zeros(y.shape[1]), np.zeros(y.shape[1]), np.zeros(y.shape[1])
            for e, w in zip(ids[t], weights[t].astype(np.float64)):
                if not 0 <= e < self.gate.count:
                    continue
                v, b = R.mlp(x[t], self.vg[e], self.vu[e], self.vd[e])
                want, bound, size = want + w * v, bound + abs(w) * b, size + np.abs(w * v)
            if residual is not None:
                want, size = want + residual[t], size + np.abs(residual[t])
            bound += (top_k + 1) * 2.0**-24 * (size + bound)  # a fused step a choice, and the residual
            assert np.all(np.abs(y[t] - want) <= bound), (t, np.abs(y[t] - want).max(), bound.min())


MLPS = [
    # type, down's, experts, tokens, top_k, hidden, ffn, residual, pad
    (H.Q4_0, H.Q4_0, 1, 1, 1, 1, 1, False, 0.0), (H.Q8_0, H.Q8_0, 2, 1, 2, 64, 96, False, 0.0),
    (H.Q4_0, H.Q8_0, 8, 1, 8, 96, 50, True, 0.0), (H.Q4_0, H.Q4_0, 8, 2, 2, 576, 130, True, 0.0),
    (H.Q8_0, H.Q4_0, 4, 8, 3, 33, 77, False, 0.2), (H.Q4_0, H.Q4_0, 64, 16, 8, 128, 64, True, 0.1),
    (H.Q8_0, H.Q8_0, 3, 100, 2, 72, 160, True, 0.1), (H.Q4_0, H.Q4_0, 6, 90, 4, 100, 36, False, 0.3),
    # Long work in the second product alone (after tiles of 16 rows), in the first, in the second, in both.
    (H.Q4_0, H.Q8_0, 64, 1000, 2, 4100, 40, True, 0.0),
    (H.Q4_0, H.Q8_0, 8, 600, 2, 64, 2080, True, 0.1), (H.Q8_0, H.Q4_0, 4, 700, 2, 2100, 40, False, 0.0),
    (H.Q4_0, H.Q4_0, 8, 1500, 2, 1040, 1100, True, 0.05),
]


@pytest.mark.parametrize("qtype,down_type,count,tokens,top_k,hidden,ffn,res,pad", MLPS)
def test_mlp(qtype, down_type, count, tokens, top_k, hidden, ffn, res, pad):
    rng = np.random.default_rng(hidden * 17 + ffn)
    layer = Layer(rng, qtype, down_type, count, hidden, ffn)
    ids = draw_ids(rng, tokens, top_k, count, pad)
    weights = rng.random((tokens, top_k)).astype(np.float32)
    weights[ids < 0] = NAN  # adds nothing, whatever its weight
    x = rng.standard_normal((tokens, hidden)).astype(np.float32)
    residual = rng.standard_normal((tokens, hidden)).astype(np.float32) if res else None
    y = layer.run(ids, weights, x, residual, pad=3)
    layer.check(y, ids, weights, x, residual)
    if res:
        again = layer.run(ids, weights, x, residual, pad=3, in_place=True)
        assert np.array_equal(y.view(np.uint32), again.view(np.uint32))


def test_mlp_same_expert_twice_and_none():
    rng = np.random.default_rng(8)
    layer = Layer(rng, H.Q4_0, H.Q4_0, 4, 64, 48)
    x = rng.standard_normal((3, 64)).astype(np.float32)
    weights = rng.random((3, 2)).astype(np.float32)
    for ids in ([[2, 2], [-1, -1], [3, 2]], [[-1, -1]] * 3, [[1, 1]] * 3, [[4, -7], [2**31 - 1, 0], [0, 4]]):
        ids = np.array(ids, np.int32)
        y = layer.run(ids, weights, x)
        layer.check(y, ids, weights, x)
        assert (y[(ids < 0).all(1)] == 0).all()


def test_layer_together():
    """Router logits by the fp32 product, the route, the MLP, added to the state: as a decoder's layer runs them."""
    rng = np.random.default_rng(31)
    hidden, ffn, count, top_k = 96, 64, 8, 2
    layer = Layer(rng, H.Q8_0, H.Q4_0, count, hidden, ffn)
    wr = rng.standard_normal((count, hidden)).astype(np.float32)
    router = H.Weight.quantize(wr, count, hidden, H.F32)
    for tokens in (1, 4, 70):
        x = rng.standard_normal((tokens, hidden)).astype(np.float32)
        xb, lb, sb = dev(x), H.DeviceBuffer(tokens * count * 4), dev(x * 2)
        ib, wb = H.DeviceBuffer(tokens * top_k * 4), H.DeviceBuffer(tokens * top_k * 4)
        work = Workspace(H.moe_mlp_bytes(layer.gate, layer.down, tokens, top_k))
        router.matmul_dev(xb.ptr, tokens, None, lb.ptr)
        H.moe_route(lb.ptr, tokens, count, top_k, ib.ptr, wb.ptr)
        H.moe_mlp(layer.gate, layer.up, layer.down, ib.ptr, wb.ptr, tokens, top_k, xb.ptr, sb.ptr, work.buf.ptr, work.n, residual=sb.ptr)
        H.synchronize()
        logits = lb.download(np.float32).reshape(tokens, count)
        ids, weights = R.route(logits, top_k, True, 1.0)
        got = wb.download(np.float32).reshape(tokens, top_k)
        assert np.array_equal(ib.download(np.int32).reshape(tokens, top_k), ids)
        assert np.all(np.abs(got - weights) <= 2.0**-24 * 100)
        layer.check(sb.download(np.float32).reshape(tokens, hidden), ids, got, x, x * 2)


@pytest.mark.parametrize("tokens,hidden,ffn", [(1, 128, 80), (6, 128, 80), (60, 128, 80), (600, 64, 2080), (2100, 48, 2080), (2100, 1100, 64)])
def test_captured_and_replayed(tokens, hidden, ffn):
    """Two graphs that share a workspace, replayed in turn with other inputs and other choices."""
    rng = np.random.default_rng(41)
    count, top_k = 8, 2
    layer = Layer(rng, H.Q4_0, H.Q4_0, count, hidden, ffn)
    lb, xb = H.DeviceBuffer(tokens * count * 4), H.DeviceBuffer(tokens * hidden * 4)
    ib, wb = H.DeviceBuffer(tokens * top_k * 4), H.DeviceBuffer(tokens * top_k * 4)
    yb, zb = H.DeviceBuffer(tokens * hidden * 4), H.DeviceBuffer(tokens * top_k * ffn * 4)
    work = Workspace(max(H.moe_mlp_bytes(layer.gate, layer.down, tokens, top_k), H.moe_matmul_bytes(layer.gate, tokens * top_k, top_k)))

    def mlp():
        H.moe_route(lb.ptr, tokens, count, top_k, ib.ptr, wb.ptr)
        H.moe_mlp(layer.gate, layer.up, layer.down, ib.ptr, wb.ptr, tokens, top_k, xb.ptr, yb.ptr, work.buf.ptr, work.n)

    def matmul():
        H.moe_matmul(layer.gate, ib.ptr, tokens * top_k, xb.ptr, zb.ptr, work.buf.ptr, work.n, per_row=top_k)

    def inputs():
        logits = rng.standard_normal((tokens, count)).astype(np.float32)
        logits[rng.random(logits.shape) < 0.2] = -INF
        lb.upload(logits)
        xb.upload(rng.standard_normal((tokens, hidden)).astype(np.float32))

    inputs()
    mlp()
    H.synchronize()
    a, b = H.Graph(mlp), H.Graph(matmul)
    for _ in range(4):
        inputs()
        zb.upload(np.zeros(tokens * top_k * ffn, np.float32))
        a.launch()
        b.launch()
        H.synchronize()
        y, z = yb.download(np.float32), zb.download(np.float32)
        mlp()
        zb.upload(np.zeros(tokens * top_k * ffn, np.float32))
        matmul()
        H.synchronize()
        assert np.array_equal(y.view(np.uint32), yb.download(np.float32).view(np.uint32))
        assert np.array_equal(z.view(np.uint32), zb.download(np.float32).view(np.uint32))


@pytest.mark.parametrize("tokens,hidden,ffn,count", [(1, 64, 48, 4), (2, 64, 48, 4), (9, 64, 48, 4), (300, 64, 48, 4), (900, 64, 2080, 4)])
def test_mlp_in_place_of_x(tokens, hidden, ffn, count):
    """y may be x, with a residual of its own or x itself as the residual."""
    rng = np.random.default_rng(51)
    layer = Layer(rng, H.Q8_0, H.Q4_0, count, hidden, ffn)
    ids = draw_ids(rng, tokens, 2, count, 0.2)
    weights = rng.random(ids.shape).astype(np.float32)
    x, r = rng.standard_normal((2, tokens, hidden)).astype(np.float32)
    ib, wb, rb = dev(ids), dev(weights), dev(r)
    work = Workspace(H.moe_mlp_bytes(layer.gate, layer.down, tokens, 2))
    for residual in (None, r, x):
        want = layer.run(ids, weights, x, residual)
        xb = dev(x)
        H.moe_mlp(layer.gate, layer.up, layer.down, ib.ptr, wb.ptr, tokens, 2, xb.ptr, xb.ptr, work.buf.ptr, work.n,
                  residual=None if residual is None else rb.ptr if residual is r else xb.ptr)
        H.synchronize()
        assert np.array_equal(xb.download(np.float32).view(np.uint32).reshape(tokens, hidden), want.view(np.uint32))
        layer.check(want, ids, weights, x, residual)


@pytest.mark.parametrize("tokens,ffn", [(1, 96), (2, 96), (7, 96), (150, 96), (700, 2080)])
@pytest.mark.parametrize("qtype", [H.Q4_0, H.Q8_0])
def test_mlp_nonfinite_rows(tokens, ffn, qtype):
    """inf and NaN of a row of x, of a weight or of the residual show in that token alone."""
    rng = np.random.default_rng(52)
    layer = Layer(rng, qtype, qtype, 4, 48, ffn)
    ids = draw_ids(rng, tokens, 2, 4)
    weights = rng.random(ids.shape).astype(np.float32) + 0.1
    x, r = rng.standard_normal((2, tokens, 48)).astype(np.float32)
    for t in (0, 3, tokens - 1):
        for kind, v in ((0, INF), (0, NAN), (1, INF), (1, NAN), (2, -INF), (2, NAN)):
            if t >= tokens:
                continue
            a = [x.copy(), weights.copy(), r.copy()]
            a[kind][t, 1] = v
            y = layer.run(ids, a[1], a[0], a[2])
            if kind == 2:
                assert np.isnan(y[t, 1]) if np.isnan(v) else y[t, 1] == v
                a[2][t, 1], y[t, 1] = 0, layer.run(ids, weights, x, np.where(np.isfinite(a[2]), a[2], 0).astype(np.float32))[t, 1]
                assert np.isfinite(y[t]).all()
            else:
                assert not np.isfinite(y[t]).any() if np.isnan(v) else not np.isfinite(y[t]).all()
                y, a[0], a[1] = y.copy(), x, weights
                y[t] = layer.run(ids, weights, x, a[2])[t]
            if tokens < 10 or t == 0:
                layer.check(y, ids, weights, x, a[2])


@pytest.mark.parametrize("tokens,ffn", [(1, 96), (5, 96), (120, 96), (700, 2080)])
def test_mlp_saturated_gates(tokens, ffn):
    """Gates from deep below 0 to far above: silu at its ends."""
    rng = np.random.default_rng(53)
    layer = Layer(rng, H.Q8_0, H.Q4_0, 4, 64, ffn)
    ids = draw_ids(rng, tokens, 2, 4)
    weights = rng.random(ids.shape).astype(np.float32)
    for size in (20.0, 100.0, 3e4):
        x = (rng.standard_normal((tokens, 64)) * size).astype(np.float32)
        layer.check(layer.run(ids, weights, x), ids, weights, x)


def test_one_workspace_for_smaller_calls():
    """The bytes for the most tokens hold every smaller call, whichever kernels that takes; nothing of one call is left for the next."""
    rng = np.random.default_rng(54)
    layer = Layer(rng, H.Q4_0, H.Q8_0, 8, 40, 2080)
    most = 2200
    work = Workspace(max(H.moe_mlp_bytes(layer.gate, layer.down, most, 2), H.moe_matmul_bytes(layer.gate, 2 * most, 2)))
    for tokens in (most, 1, 700, 2, 64, 3, 300, 1000, 9):
        ids = draw_ids(rng, tokens, 2, 8, 0.2)
        weights = rng.random(ids.shape).astype(np.float32)
        x = rng.standard_normal((tokens, 40)).astype(np.float32)
        ib, wb, xb, yb, zb = dev(ids), dev(weights), dev(x), H.DeviceBuffer(tokens * 160), dev(np.full((tokens * 2, 2080), GUARD, np.float32))
        H.moe_mlp(layer.gate, layer.up, layer.down, ib.ptr, wb.ptr, tokens, 2, xb.ptr, yb.ptr, work.buf.ptr, work.n)
        H.moe_matmul(layer.gate, ib.ptr, tokens * 2, xb.ptr, zb.ptr, work.buf.ptr, work.n, per_row=2)
        H.synchronize()
        work.intact()
        layer.check(yb.download(np.float32).reshape(tokens, 40), ids, weights, x)
        check_matmul(zb.download(np.float32).reshape(tokens * 2, 2080), ids, x, 2, layer.vg)


@pytest.mark.parametrize("per_row", [2**31 - 1, 2**31, 2**32, 2**32 + 1, 2**64 - 1])
@pytest.mark.parametrize("slots,out", [(5, 40), (70, 40), (1300, 4100)])
def test_matmul_one_row_for_all(per_row, slots, out):
    """More slots a row than there are, beyond 32 bits too: the one row of x."""
    rng = np.random.default_rng(55)
    experts, values = make(rng, H.Q4_0, 2, out, 64)
    ids = rng.integers(-1, 2, slots).astype(np.int32)
    x = rng.standard_normal((1, 64)).astype(np.float32)
    check_matmul(run_matmul(experts, ids, x, per_row), ids, x, per_row, values)


@pytest.mark.parametrize("slots,out", [(12, 40), (150, 40), (1300, 4100)])
@pytest.mark.parametrize("qtype", [H.Q4_0, H.Q8_0])
def test_matmul_rows_apart(slots, out, qtype):
    """A row's bits do not depend on what stands in the others, nor on their experts."""
    rng = np.random.default_rng(58)
    experts, _ = make(rng, qtype, 5, out, 100)
    ids = rng.integers(0, 5, slots).astype(np.int32)
    x = rng.standard_normal((slots, 100)).astype(np.float32)
    keep = rng.permutation(slots)[:slots // 4]
    first = run_matmul(experts, ids, x, 1)
    others = np.setdiff1d(np.arange(slots), keep)
    ids[others] = rng.integers(-1, 5, len(others))
    x[others] = (rng.standard_normal((len(others), 100)) * 1e6).astype(np.float32)
    x[others[::3]] = NAN
    again = run_matmul(experts, ids, x, 1)
    assert np.array_equal(first[keep].view(np.uint32), again[keep].view(np.uint32))


@pytest.mark.parametrize("tokens,ffn", [(5, 96), (150, 96), (900, 2080)])
def test_mlp_tokens_apart(tokens, ffn):
    """Nor does a token's MLP, of three tokens or more."""
    rng = np.random.default_rng(59)
    layer = Layer(rng, H.Q4_0, H.Q8_0, 5, 64, ffn)
    ids, weights = draw_ids(rng, tokens, 2, 5), rng.random((tokens, 2)).astype(np.float32)
    x = rng.standard_normal((tokens, 64)).astype(np.float32)
    keep = rng.permutation(tokens)[:(tokens + 3) // 4]
    first = layer.run(ids, weights, x)
    others = np.setdiff1d(np.arange(tokens), keep)
    ids[others], weights[others] = draw_ids(rng, len(others), 2, 5, 0.3), INF
    x[others] = (rng.standard_normal((len(others), 64)) * 1e6).astype(np.float32)
    again = layer.run(ids, weights, x)
    assert np.array_equal(first[keep].view(np.uint32), again[keep].view(np.uint32))


def put(at, a):
    H.check(H.load().llmi_hip_memcpy_h2d(at, a.ctypes.data_as(C.c_void_p), a.nbytes))


@pytest.mark.parametrize("slots", [3, 100])
def test_experts_past_four_gigabytes(slots):
    """The last of 4096 experts whose codes end past 2^32 bytes; what the others hold is left as it came."""
    rng = np.random.default_rng(61)
    count, out, n_in = 4096, 64, 16384
    data, scales, values = R.matrices(rng, H.Q8_0, 2, out, n_in)
    d, s = H.DeviceBuffer(count * data[0].nbytes), H.DeviceBuffer(count * scales[0].nbytes)
    where = {4095: 0, 2050: 1}
    for e, i in where.items():
        put(d.ptr + e * data[0].nbytes, data[i])
        put(s.ptr + e * scales[0].nbytes, scales[i])
    experts = H.Experts.upload_dev(d.ptr, s.ptr, count, out, n_in, H.Q8_0)
    ids = np.where(np.arange(slots) % 3 == 0, 4095, np.where(np.arange(slots) % 3 == 1, 2050, -1)).astype(np.int32)
    x = rng.standard_normal((slots, n_in)).astype(np.float32)
    y = run_matmul(experts, ids, x, 1)
    for r in range(slots):
        if ids[r] < 0:
            assert (y[r] == GUARD).all()
            continue
        want, bound = R.product(x[r], values[where[ids[r]]])
        assert np.all(np.abs(y[r] - want) <= bound), r


@pytest.mark.parametrize("slots,out,stride", [(3, 40, 1 << 29), (70, 40, 1 << 25), (1300, 4100, 1 << 20)])
def test_rows_past_four_gigabytes(slots, out, stride):
    """Rows of x and y so far apart that the last ones begin past 2^32 bytes."""
    rng = np.random.default_rng(62)
    experts, values = make(rng, H.Q4_0, 2, out, 100)
    ids = rng.integers(0, 2, slots).astype(np.int32)
    x = rng.standard_normal((slots, 100)).astype(np.float32)
    xb, yb, ib = H.DeviceBuffer(slots * stride * 4), H.DeviceBuffer(slots * stride * 4), dev(ids)
    for r in range(slots):
        put(xb.ptr + r * stride * 4, x[r])
    work = Workspace(H.moe_matmul_bytes(experts, slots, 1))
    H.moe_matmul(experts, ib.ptr, slots, xb.ptr, yb.ptr, work.buf.ptr, work.n, x_stride=stride, y_stride=stride)
    H.synchronize()
    work.intact()
    y = np.zeros((slots, out), np.float32)
    for r in range(slots):
        H.check(H.load().llmi_hip_memcpy_d2h(y[r].ctypes.data_as(C.c_void_p), yb.ptr + r * stride * 4, out * 4))
    check_matmul(y, ids, x, 1, values)


def test_two_streams_at_once():
    """Calls on two streams of the caller's, with a workspace each: the results of each alone."""
    create = H.load().hipStreamCreateWithFlags  # found through the library's own dependencies
    rng = np.random.default_rng(56)
    layer = Layer(rng, H.Q4_0, H.Q8_0, 8, 64, 2080)
    streams, calls = [], []
    for tokens in (700, 40, 1, 2100):
        ids = draw_ids(rng, tokens, 2, 8, 0.1)
        weights = rng.random(ids.shape).astype(np.float32)
        x = rng.standard_normal((tokens, 64)).astype(np.float32)
        want = layer.run(ids, weights, x)
        layer.check(want, ids, weights, x)
        work = Workspace(H.moe_mlp_bytes(layer.gate, layer.down, tokens, 2))
        calls.append((tokens, dev(ids), dev(weights), dev(x), dev(np.zeros_like(x)), work, want))
    for _ in range(2):
        s = C.c_void_p()
        assert create(C.byref(s), 1) == 0  # non-blocking
        streams.append(s.value)
    H.synchronize()
    for _ in range(5):
        for i, (tokens, ib, wb, xb, yb, work, _) in enumerate(calls):
            H.moe_mlp(layer.gate, layer.up, layer.down, ib.ptr, wb.ptr, tokens, 2, xb.ptr, yb.ptr, work.buf.ptr, work.n, stream=streams[i % 2])
    for s in streams:
        assert H.load().hipStreamSynchronize(C.c_void_p(s)) == 0
    for tokens, *_, yb, work, want in calls:
        work.intact()
        assert np.array_equal(yb.download(np.float32).reshape(want.shape).view(np.uint32), want.view(np.uint32))
    for s in streams:
        assert H.load().hipStreamDestroy(C.c_void_p(s)) == 0


def test_route_on_a_stream_and_repeated():
    """The router on a stream of the caller's, many tokens, twice: the same bits."""
    create = H.load().hipStreamCreateWithFlags
    rng = np.random.default_rng(57)
    logits = rng.standard_normal((20000, 60)).astype(np.float32)
    lb = dev(logits)
    s = C.c_void_p()
    assert create(C.byref(s), 1) == 0
    got = []
    for _ in range(2):
        ib, wb = dev(np.zeros((20000, 4), np.int32)), dev(np.zeros((20000, 4), np.float32))
        H.moe_route(lb.ptr, 20000, 60, 4, ib.ptr, wb.ptr, stream=s.value)
        assert H.load().hipStreamSynchronize(s) == 0
        got.append((ib.download(np.int32).reshape(-1, 4), wb.download(np.float32).reshape(-1, 4)))
    assert np.array_equal(got[0][0], got[1][0]) and np.array_equal(got[0][1].view(np.uint32), got[1][1].view(np.uint32))
    some_rows = np.arange(0, 20000, 97)
    ids, w = R.route(logits[some_rows], 4, True, 1.0)
    assert np.array_equal(got[0][0][some_rows], ids) and np.all(np.abs(got[0][1][some_rows] - w) <= w * 2.0**-24 * 80)
    assert H.load().hipStreamDestroy(s) == 0


# ---------------------------------------------------------------- refusals


def test_refusals():
    rng = np.random.default_rng(1)
    data, scales, _ = R.matrices(rng, H.Q4_0, 2, 8, 32)
    d, s = dev(data), dev(scales)

    def refused(why, fn, *a, **k):
        with pytest.raises(H.HipError, match=why):
            fn(*a, **k)

    for args, why in (((0, 8, 32, H.Q4_0), "experts"), ((4097, 8, 32, H.Q4_0), "experts"), ((2, 0, 32, H.Q4_0), "in and out"),
                      ((2, 8, 0, H.Q4_0), "in and out"), ((2, 8, 2**18 + 1, H.Q4_0), "in and out"), ((2, 8, 32, H.F32), "type")):
        refused(why, H.Experts.upload_dev, d.ptr, s.ptr, *args)
    refused("null", H.Experts.upload_dev, None, s.ptr, 2, 8, 32, H.Q4_0)
    w = [H.Weight.upload(data[0], scales[0], 8, 32, H.Q4_0), H.Weight.upload(data[0, :4], scales[0, :4], 4, 32, H.Q4_0)]
    refused("different", H.Experts.from_weights, w)
    refused("type", H.Experts.from_weights, [H.Weight.quantize(np.zeros((8, 32), np.float32), 8, 32, H.F32)])
    gate = H.Experts.upload_dev(d.ptr, s.ptr, 2, 8, 32, H.Q4_0)
    other = make(rng, H.Q8_0, 2, 8, 32)[0]
    down = make(rng, H.Q8_0, 2, 32, 8)[0]
    buf = H.DeviceBuffer(1 << 16)
    p = buf.ptr
    refused("at least 1", H.moe_matmul_bytes, gate, 4, 0)
    refused("2\\^24", H.moe_matmul_bytes, gate, 2**24 + 1)
    n = H.moe_matmul_bytes(gate, 4)
    refused("needed", H.moe_matmul, gate, p, 4, p, p + 4096, p, n - 1)
    refused("aligned", H.moe_matmul, gate, p, 4, p, p + 4096, p + 8, n)
    y = p + 4096
    refused("y must not be x", H.moe_matmul, gate, p, 4, p, p, p, n)
    refused("null", H.moe_matmul, gate, None, 4, p, y, p, n)
    refused("null", H.moe_matmul, gate, p, 4, None, p, p, n)
    refused("null", H.moe_matmul, gate, p, 4, p, None, p, n)
    refused("null", H.moe_matmul, gate, p, 4, p, p + 4096, None, n)
    refused("stride", H.moe_matmul, gate, p, 4, p, p + 4096, p, n, x_stride=31)
    refused("stride", H.moe_matmul, gate, p, 4, p, p + 4096, p, n, y_stride=7)
    n = H.moe_mlp_bytes(gate, down, 2, 2)
    mlp = dict(ids=p, weights=p, tokens=2, top_k=2, x=p, y=p, work=p, work_bytes=n)
    refused("different types", H.moe_mlp, gate, other, down, **mlp)
    refused("down's", H.moe_mlp, gate, gate, gate, **mlp)
    refused("down's", H.moe_mlp_bytes, gate, gate, 2, 2)
    for change, why in ((dict(top_k=0), "top_k"), (dict(top_k=65), "top_k"), (dict(tokens=2**24), "2\\^24"), (dict(work_bytes=n - 1), "needed"),
                        (dict(work=p + 4), "aligned"), (dict(ids=None), "null"), (dict(weights=None), "null"), (dict(x=None), "null"),
                        (dict(y=None), "null"), (dict(work=None), "null"), (dict(x_stride=31), "stride"), (dict(y_stride=31), "stride"),
                        (dict(residual=p, residual_stride=31), "stride"), (dict(residual=p, residual_stride=40), "in place")):
        refused(why, H.moe_mlp, gate, gate, down, **dict(mlp, **change))
    for args, why in (((4, 0, 1), "experts"), ((4, 1025, 1), "experts"), ((4, 8, 0), "top_k"), ((4, 8, 9), "top_k"), ((4, 100, 65), "top_k"),
                      ((2**24 + 1, 8, 2), "2\\^24")):
        refused(why, H.moe_route, p, *args, p, p)
    refused("stride", H.moe_route, p, 4, 8, 2, p, p, stride=7)
    refused("finite", H.moe_route, p, 4, 8, 2, p, p, scale=float("inf"))
    for null in range(3):
        a = [p, p, p]
        a[null] = None
        refused("null", H.moe_route, a[0], 4, 8, 2, a[1], a[2])
    # Nothing to do: no pointers needed.
    H.moe_route(None, 0, 8, 2, None, None)
    H.moe_matmul(gate, None, 0, None, None, None, 0)
    H.moe_mlp(gate, gate, down, None, None, 0, 2, None, None, None, 0)
