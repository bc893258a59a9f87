"""The paged 8-bit key/value cache in 64 bits, from its definition: what the
GPU tests compare llmi_hip_kv8_* with."""

import numpy as np

BLOCK = 16


def turn(x, w, eps, cos, sin):
    """Norm and rotation of rows [..., dim] in 64 bits (w, cos, sin may be None)."""
    x = np.asarray(x, dtype=np.float64)
    if w is not None:
        x = x / np.sqrt((x * x).mean(-1, keepdims=True) + np.float64(np.float32(eps))) * w.astype(np.float64)
    if cos is not None:
        a, b = np.split(x, 2, -1)
        c, s = cos.astype(np.float64), sin.astype(np.float64)
        x = np.concatenate([a * c - b * s, b * c + a * s], -1)
    return x


def quantize(rows):
    """fp32 rows [n][kv][dim] as the cache holds them: 64-bit values code * scale (the last block as far as it goes)."""
    out = np.zeros(rows.shape, dtype=np.float64)
    for b in range(0, len(rows), BLOCK):
        x = rows[b:b + BLOCK].astype(np.float64)
        with np.errstate(invalid="ignore", divide="ignore", over="ignore"):
            top = np.abs(x).max((0, 2))
            scale = (top / 127.0).astype(np.float32).astype(np.float64)[None, :, None]
            codes = np.clip(np.rint(x / np.where(scale > 0, scale, 1.0)), -127, 127)
            out[b:b + BLOCK] = np.where(np.isfinite(scale), np.where(scale > 0, codes, 0.0) * scale, np.nan)
    return out


def attend(q, k, v, start, scale):
    """q [n][heads][dim] at positions start.. over k, v [len][kv][dim], causal, in 64 bits."""
    n, heads, dim = q.shape
    group = heads // k.shape[1]
    kk, vv = np.repeat(k, group, 1), np.repeat(v, group, 1)
    out = np.zeros((n, heads, dim))
    for i in range(n):
        m = start + i + 1
        s = np.einsum("hd,jhd->hj", q[i].astype(np.float64), kk[:m]) * scale
        p = np.exp(s - s.max(1, keepdims=True))
        out[i] = np.einsum("hj,jhd->hd", p / p.sum(1, keepdims=True), vv[:m])
    return out


def attend_bound(q, k, v, scale):
    """How far fp32 sums may be off: each score by (dim + 4) roundings of its
    terms, each weight by twice that and an exponential of two roundings, and
    the weighted sum by a rounding per term of a 64-position tile and per tile."""
    dim, n = q.shape[-1], len(k)
    group = q.shape[1] // k.shape[1]
    top = np.abs(np.nan_to_num(k)).max(0)  # [kv][dim]
    score = abs(scale) * np.einsum("nhd,hd->nh", np.abs(q), np.repeat(top, group, 0)).max()
    return float(np.abs(np.nan_to_num(v)).max()) * (2 * score * (dim + 4) * 2.0**-24 + (dim + 64 + n / 64) * 2.0**-23)


def tables(rng, lens, page, spare=3):
    """Random page tables for sequences of these lengths: (tables, pages of the pool)."""
    per = [-(-n // page) for n in lens]
    pages = sum(per) + spare
    order = rng.permutation(pages)
    out = np.zeros((len(lens), max(per + [1])), dtype=np.int32)
    at = 0
    for i, n in enumerate(per):
        out[i, :n] = order[at:at + n]
        at += n
    return out, pages


def rope(positions, dim, theta=10000.0):
    angle = np.arange(positions)[:, None] * theta ** (-np.arange(0, dim, 2) / dim)
    return np.cos(angle).astype(np.float32), np.sin(angle).astype(np.float32)


def pack(k, v, tables, lens, page, pages, rng):
    """int8 codes k, v [sequence][len][kv][dim] (lists) in the pool's layout; unused places are random."""
    kv, dim = k[0].shape[1:]
    shape = (pages, kv, page // BLOCK, dim // 16, 16, 16)
    pk, pv = (rng.integers(-128, 128, shape, dtype=np.int8) for _ in range(2))
    for i, n in enumerate(lens):
        pos = np.arange(n)
        at = (tables[i, pos // page], slice(None), pos % page // BLOCK)
        pk[at[0], :, at[2], :, pos % BLOCK] = k[i].reshape(n, kv, dim // 16, 16)
        pv[at[0], :, at[2], :, :, pos % BLOCK] = v[i].reshape(n, kv, dim // 16, 16)
    return pk, pv
