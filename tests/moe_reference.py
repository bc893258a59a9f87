"""A layer of experts in 64 bits, from its definition, and how far fp32 sums
may be off: what the tests compare llmi_hip_moe_* with."""

import numpy as np

BLOCK = 32
Q8_0, Q4_0 = 1, 2


def matrices(rng, qtype, count, out, n_in, spread=1.0):
    """Random planar codes and scales of `count` experts, and their values in 64 bits [count][out][in]."""
    blocks = -(-n_in // BLOCK)
    scales = (np.exp(spread * rng.standard_normal((count, out, blocks))) / np.sqrt(n_in)).astype(np.float32)
    if qtype == Q8_0:
        codes = rng.integers(-127, 128, (count, out, n_in), dtype=np.int8)
        scales /= np.float32(64)
        data = codes.view(np.uint8)
    else:
        codes = rng.integers(-8, 8, (count, out, n_in), dtype=np.int8)
        scales /= np.float32(4)
        nib = (codes + 8).astype(np.uint8)
        if n_in % 2:  # the last byte's high half means nothing
            nib = np.concatenate([nib, rng.integers(0, 16, (count, out, 1), dtype=np.uint8)], -1)
        data = nib[..., 0::2] | nib[..., 1::2] << 4
    values = codes.astype(np.float64) * np.repeat(scales.astype(np.float64), BLOCK, -1)[..., :n_in]
    return np.ascontiguousarray(data), scales, values


def route(logits, top_k, renormalise, scale):
    """(ids, weights in 64 bits) by sorting (falling logit, rising index)."""
    l = np.asarray(logits, dtype=np.float64)
    ids = np.full((len(l), top_k), -1, np.int32)
    weights = np.zeros((len(l), top_k))
    for t, row in enumerate(l):
        live = np.nonzero(row > -np.inf)[0]  # NaN compares false
        if len(live) == 0:
            continue
        top = row[live].max()
        with np.errstate(invalid="ignore"):
            p = np.where(row[live] == top, 1.0, np.exp(row[live] - top))
        best = sorted(range(len(live)), key=lambda i: (-row[live[i]], live[i]))[:top_k]
        total = p[best].sum() if renormalise else p.sum()
        ids[t, :len(best)] = live[best]
        weights[t, :len(best)] = scale * p[best] / total
    return ids, weights


def product(x, w):
    """x [in] against w [out][in], and the bound of an fp32 evaluation: every
    element of x is off by 2^-22 of itself (its two 11-bit roundings) or by
    2^-39 of the row's largest, a code's product and its sums take part in at
    most 32 additions of the block, one product with the scale and one
    addition a block, each off by 2^-24 of what it gives, which the sum of
    magnitudes bounds; matrix instructions may cut where others round: twice."""
    x = np.asarray(x, dtype=np.float64)
    size = np.abs(w) @ np.abs(x)
    blocks = -(-len(x) // BLOCK)
    steps = 2 * 32 + 2 * (blocks + 2)
    top = np.abs(x).max() if len(x) else 0.0
    return w @ x, size * (2.0**-22 + steps * 2.0**-23) + np.abs(w).sum(1) * top * 2.0**-39


def silu(g):
    with np.errstate(over="ignore"):
        return g / (1.0 + np.exp(-g))


def mlp(x, gate, up, down):
    """One expert's MLP of one row with its bound: the gate's and up's errors
    through silu (slope at most 1.1) and the product, an exponential and three
    roundings (8 units), then the second product of a vector known that well."""
    g, dg = product(x, gate)
    u, du = product(x, up)
    h = silu(g) * u
    dh = 1.1 * dg * (np.abs(u) + du) + np.abs(silu(g)) * du + 8 * 2.0**-24 * np.abs(h)
    y, dy = product(h, down)
    return y, dy * 1.01 + np.abs(down) @ dh
