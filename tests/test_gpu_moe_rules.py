"""Calls of a layer of experts whose operands overlap, and such as lie close
together and do not."""

import numpy as np
import pytest

import llmi_hip as H
import moe_reference as R
import test_gpu_moe as G

pytestmark = pytest.mark.gpu


def refused(fn, *a, **k):
    with pytest.raises(H.HipError, match="overlaps"):
        fn(*a, **k)


@pytest.mark.parametrize("slots", [4, 150])
def test_matmul_operands_apart(slots):
    rng = np.random.default_rng(1)
    experts, values = G.make(rng, H.Q8_0, 3, 40, 64)
    n = H.moe_matmul_bytes(experts, slots)
    ids = rng.integers(-1, 3, slots).astype(np.int32)
    x = rng.standard_normal((slots, 64)).astype(np.float32)
    # One allocation: rows of x and, beside them, of y (stride 128), ids, workspace.
    rows, at_ids = slots * 512, slots * 512 + 4
    at_work = (at_ids + slots * 4 + 255) // 256 * 256
    buf = H.DeviceBuffer(at_work + n)
    p = buf.ptr
    y = np.full((slots, 128), G.GUARD, np.float32)
    y[:, :64] = x
    G.put(p, y)
    G.put(p + at_ids, ids)

    def call(xp, yp, ip, wp, xs=128, ys=128):
        H.moe_matmul(experts, ip, slots, xp, yp, wp, n, x_stride=xs, y_stride=ys)

    good = (p, p + 256, p + at_ids, p + at_work)
    for change in ((0, p + 4), (0, p + at_work + 256), (1, p + 252), (1, p + 4), (1, p + at_ids - 100), (1, p + at_work + n - 4),
                   (2, p + 256), (2, p + at_work + n - 4), (3, p), (3, p + rows - 512), (3, p + at_ids // 256 * 256)):
        refused(call, *(change[1] if i == change[0] else v for i, v in enumerate(good)))
    refused(call, *good, ys=100)
    refused(call, *good, xs=64)
    H.synchronize()
    assert np.array_equal(buf.download(np.float32)[:slots * 128].reshape(slots, 128).view(np.uint32), y.view(np.uint32))
    call(*good)
    H.synchronize()
    got = buf.download(np.float32)[:slots * 128].reshape(slots, 128)
    assert np.array_equal(got[:, :64], x) and (got[:, 104:] == G.GUARD).all()
    G.check_matmul(got[:, 64:104], ids, x, 1, values)


@pytest.mark.parametrize("tokens", [1, 2, 50])
def test_mlp_operands_apart(tokens):
    rng = np.random.default_rng(2)
    layer = G.Layer(rng, H.Q4_0, H.Q8_0, 4, 32, 48)
    n = H.moe_mlp_bytes(layer.gate, layer.down, tokens, 2)
    ids, weights = G.draw_ids(rng, tokens, 2, 4), rng.random((tokens, 2)).astype(np.float32)
    x, r = rng.standard_normal((2, tokens, 32)).astype(np.float32)
    want = layer.run(ids, weights, x, r)
    at_work = tokens * 256
    buf = H.DeviceBuffer(at_work + n)
    p, ib, wb, xb = buf.ptr, G.dev(ids), G.dev(weights), G.dev(x)
    both = np.concatenate([r, np.zeros_like(r)], 1)  # the residual's rows, y's beside them
    G.put(p, both)

    def call(y, residual, ids=ib.ptr, weights=wb.ptr, work=p + at_work, x=xb.ptr, x_stride=32, stride=64):
        H.moe_mlp(layer.gate, layer.up, layer.down, ids, weights, tokens, 2, x, y, work, n, residual=residual, x_stride=x_stride,
                  residual_stride=64, y_stride=stride)

    y = p + 128
    for bad in (dict(residual=p + 4), dict(residual=p + 252), dict(residual=p + at_work + n - 128), dict(ids=p + 128), dict(weights=p + 132),
                dict(work=p), dict(work=p + at_work - 256), dict(ids=p + at_work + 64), dict(weights=p + at_work + n - 4),
                dict(x=p + at_work), dict(y=p + at_work)):
        refused(call, **dict(dict(y=y, residual=p), **bad))
    if tokens > 1:
        refused(call, y, p, stride=40)
    H.synchronize()
    assert np.array_equal(buf.download(np.float32)[:tokens * 64].reshape(tokens, 64), both)
    call(y, p)
    H.synchronize()
    assert np.array_equal(buf.download(np.float32)[:tokens * 64].reshape(tokens, 64)[:, 32:].view(np.uint32), want.view(np.uint32))
    # x is free to lie under y.
    G.put(p, np.concatenate([r, x], 1))
    for shift in (0, 4, -8):
        x2 = np.zeros(tokens * 64 + 64, np.float32)
        at = 40 + shift
        for t in range(tokens):
            x2[at + t * 64:at + t * 64 + 32] = x[t]
        free = G.dev(x2)
        call(free.ptr + 160, p, x=free.ptr + 4 * at, x_stride=64)
        H.synchronize()
        got = free.download(np.float32)[40:][:tokens * 64]
        got = np.stack([got[t * 64:t * 64 + 32] for t in range(tokens)])
        assert np.array_equal(got.view(np.uint32), want.view(np.uint32))


def test_route_operands_apart():
    rng = np.random.default_rng(3)
    tokens, experts = 9, 12
    logits = rng.standard_normal((tokens, 20)).astype(np.float32)
    buf = H.DeviceBuffer(8192)
    p = buf.ptr
    G.put(p, logits)

    def call(l, i, w):
        H.moe_route(l, tokens, experts, 2, i, w, stride=20)

    for bad in ((p, p + 40, p + 4096), (p, p + 4096, p + 684), (p, p + 2048, p + 2048 + 68), (p, p + 2048, p + 2048 - 68), (p, p + 2048, p + 2048)):
        refused(call, *bad)
    H.synchronize()
    assert np.array_equal(buf.download(np.float32)[:tokens * 20].reshape(tokens, 20), logits)
    call(p, p + 2048, p + 2048 + 72)
    H.synchronize()
    ids, _ = R.route(logits[:, :experts], 2, True, 1.0)
    assert np.array_equal(buf.download(np.int32)[512:512 + 18].reshape(tokens, 2), ids)
