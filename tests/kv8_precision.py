"""Inputs for which the paged 8-bit cache's attention can be off by few
roundings only, and how many: what holds the kernels to the 22 bits of q and
of the weights that their interface promises.

Every row of q has one number that is not 0, so that a score is one product,
and the histories are short, so that the sums have few terms."""

import numpy as np

import kv8_reference as R

# heads, kv, dim, start, count: up to 64 rows (tokens x heads / kv), and more.
SHAPES = [(4, 2, 64, 30, 1), (2, 1, 128, 20, 8), (8, 1, 256, 33, 2), (12, 4, 96, 18, 5),
          (16, 1, 64, 20, 6), (40, 2, 128, 24, 4), (10, 1, 96, 15, 8), (9, 1, 256, 30, 8)]
SCALE = 0.3


def inputs(heads, kv, dim, start, count, largest):
    """(q, k, v) in fp32, scores up to about `largest`."""
    rng = np.random.default_rng(heads * 1009 + dim + int(10 * largest))
    n = start + count
    k, v = (rng.uniform(-1, 1, (n, kv, dim)).astype(np.float32) for _ in range(2))
    q = np.zeros((count, heads, dim), np.float32)
    t, h = np.meshgrid(np.arange(count), np.arange(heads), indexing="ij")
    q[t, h, rng.integers(0, dim, (count, heads))] = rng.uniform(0.5, 1, (count, heads)) * rng.choice([-1, 1], (count, heads)) * largest / SCALE
    return q, k, v


def attend(q, k, v, start, cut_q=None, cut_w=None):
    """The attention in 64 bits, with q or the weights rounded to so many bits."""
    q = q.astype(np.float64) if cut_q is None else cut(q, cut_q)
    group = q.shape[1] // k.shape[1]
    kk, vv = np.repeat(k, group, 1), np.repeat(v, group, 1)
    out = np.zeros(q.shape)
    for i in range(len(q)):
        m = start + i + 1
        s = SCALE * np.einsum("hd,jhd->hj", q[i], kk[:m])
        w = np.exp(s - s.max(1, keepdims=True))
        total = w.sum(1, keepdims=True)
        out[i] = np.einsum("hj,jhd->hd", w if cut_w is None else cut(w, cut_w), vv[:m]) / total
    return out


def cut(x, bits):
    m, e = np.frexp(np.asarray(x, dtype=np.float64))
    return np.ldexp(np.rint(m * 2.0**bits), e - bits)


def bound(q, k, v, start):
    """[count][heads][1]: in roundings of 2^-24.  A score of size s: q to 22
    bits 4, its two parts' sum or the digits' 3, the factor's three products
    and log2 e 4, the product 1, so 12 s.  In the exponent of 2, with S = s
    log2 e: the block's offset (up to S + 10) and the argument (up to 2 S + 10),
    so ln 2 (3 S + 20).  A weight: the exponential 2, its parts or digits 4.
    Each of these in the sum of weights and in that of values.  The sums: n
    weights, n values in two parts, so 3 n; the value scales' logarithms and
    the last factors 16.  All times the largest value."""
    largest = np.abs(v).max()
    group = q.shape[1] // k.shape[1]
    out = np.zeros(q.shape[:2] + (1,))
    for i in range(len(q)):
        n = start + i + 1
        s = SCALE * np.abs(np.einsum("hd,jhd->hj", q[i].astype(np.float64), np.repeat(k, group, 1)[:n])).max(1)
        weight = 12 * s + np.log(2) * (3 * s / np.log(2) + 20) + 6
        out[i, :, 0] = (2 * weight + 3 * n + 16) * 2.0**-24 * largest
    return out


def case(shape, largest):
    """q, the cache's keys and values in 64 bits, fp32 k and v, start."""
    q, k, v = inputs(*shape, largest)
    return q, R.quantize(k), R.quantize(v), k, v, shape[3]
