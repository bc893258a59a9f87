"""Calls of llmi_hip_moe_matmul_dev and _mlp_dev for each of their kernels,
with the rows of a group that csrc/moe_plan.hpp gives them, and the 64-bit
results of all rows of a call at a time (moe_reference.py has the formulas and
the bounds of one)."""

import numpy as np

import moe_reference as R

Q8_0, Q4_0 = R.Q8_0, R.Q4_0

# experts, tokens, top_k, in, out, per_row, skew of the choices; rows, grouping
MATMULS = [
    # Groups of 32 rows: each wavefront a fourth of the steps, 16 of them, 10
    # (3, 3, 3, 1), 5 (2, 2, 1, 0) and 1.
    ((13, 333, 3, 1000, 777, 3, 1.0), (32, "self")), ((8, 900, 1, 577, 1030, 1, 1.0), (32, "self")),
    ((4, 800, 2, 300, 700, 1, 1.0), (32, "self")), ((4, 1000, 2, 64, 513, 2, 1.0), (32, "self")),
    # More than eight groups of one expert, others of one or none.
    ((6, 900, 2, 200, 700, 2, 4.0), (32, "self")),
    # Rows brought in behind the grouping, by one workgroup and by several.
    ((16, 1050, 2, 840, 384, 2, 1.0), (32, "tiles")), ((8, 2400, 2, 130, 300, 1, 3.0), (32, "tiles")),
    # Groups of 64 rows; even and odd numbers of steps, two of them, one.
    ((3, 1300, 1, 900, 4100, 1, 1.0), (64, "rows")), ((3, 650, 2, 330, 4090, 2, 1.0), (64, "rows")),
    ((5, 1300, 1, 448, 2200, 1, 4.0), (64, "rows")), ((4, 1000, 1, 128, 4112, 1, 1.0), (64, "rows")),
    ((4, 4500, 1, 257, 1030, 1, 1.0), (64, "rows")), ((4, 1000, 1, 50, 4112, 1, 1.0), (64, "rows")),
    # Groups of 16, several steps a wavefront.
    ((13, 60, 3, 1300, 130, 3, 1.0), (16, "self")), ((40, 1200, 2, 700, 48, 2, 2.0), (16, "tiles")),
    ((300, 400, 4, 577, 70, 4, 1.0), (16, "tiles")),
]

# experts, tokens, top_k, hidden, ffn, skew; rows of both products, grouping.
# The steps of the products are ceil(hidden / 64) and ceil(ffn / 64).
MLPS = [
    ((16, 100, 3, 600, 130, 1.0), (16, 16, "self")), ((16, 763, 3, 600, 130, 2.0), (16, 16, "tiles")),
    ((4, 1014, 2, 1040, 130, 1.0), (16, 64, "self")), ((8, 1300, 2, 900, 64, 3.0), (16, 64, "tiles")),
    ((4, 751, 1, 450, 580, 1.0), (32, 16, "self")), ((4, 995, 3, 200, 130, 1.0), (32, 16, "tiles")),
    ((6, 673, 2, 777, 580, 1.0), (32, 32, "self")), ((4, 689, 3, 450, 200, 2.0), (32, 32, "tiles")),
    ((4, 661, 3, 1040, 200, 1.0), (32, 64, "self")), ((6, 1337, 2, 777, 330, 1.0), (32, 64, "tiles")),
    ((4, 500, 3, 200, 2080, 1.0), (64, 16, "rows")),
    ((4, 789, 2, 450, 700, 1.0), (64, 32, "rows")), ((6, 1006, 3, 320, 1500, 1.0), (64, 32, "rows")),
    ((4, 1322, 2, 777, 450, 1.0), (64, 64, "rows")), ((8, 1067, 2, 1040, 1100, 3.0), (64, 64, "rows")),
    # Calls without a grouping: a token's experts in one sum, in parts of it, two tokens.
    ((8, 1, 4, 2100, 330, 1.0), ("few",)), ((8, 1, 4, 300, 330, 1.0), ("few",)), ((8, 2, 8, 200, 2080, 1.0), ("few",)),
]


def products(x, w):
    """moe_reference.product of every row of x [rows][in]."""
    x, size = np.asarray(x, np.float64), np.abs(w)
    blocks = -(-x.shape[1] // R.BLOCK)
    steps = 2 * 32 + 2 * (blocks + 2)
    bound = (np.abs(x) @ size.T) * (2.0**-22 + steps * 2.0**-23) + np.abs(x).max(1)[:, None] * size.sum(1) * 2.0**-39
    return x @ w.T, bound


def mlps(x, gate, up, down):
    """moe_reference.mlp of every row of x."""
    g, dg = products(x, gate)
    u, du = products(x, up)
    h = R.silu(g) * u
    dh = 1.1 * dg * (np.abs(u) + du) + np.abs(R.silu(g)) * du + 8 * 2.0**-24 * np.abs(h)
    y, dy = products(h, down)
    return y, dy * 1.01 + dh @ np.abs(down).T


def sums(ids, weights, x, gate, up, down):
    """Every token's sum with its bound: a fused step a choice besides the MLPs' own."""
    tokens, top_k = ids.shape
    want, bound, size = np.zeros((3, tokens, down.shape[1]))
    for e in range(len(gate)):
        t, j = np.nonzero(ids == e)
        if len(t):
            y, b = mlps(x[t], gate[e], up[e], down[e])
            w = weights[t, j].astype(np.float64)[:, None]
            np.add.at(want, t, w * y)
            np.add.at(bound, t, np.abs(w) * b)
            np.add.at(size, t, np.abs(w * y))
    return want, bound + (top_k + 1) * 2.0**-24 * (size + bound)


def draw_ids(rng, tokens, top_k, count, pad, skew):
    p = rng.standard_normal((tokens, count)) + skew * rng.standard_normal(count)
    ids = np.argsort(-p, 1)[:, :top_k].astype(np.int32)
    ids[rng.random(ids.shape) < pad] = -1
    return ids


# ------------------------------------------- results that the second part makes


def planar(codes, qtype):
    """Codes [..][in] as rows of planar bytes."""
    if qtype == Q8_0:
        return codes.view(np.uint8)
    nib = (codes + 8).astype(np.uint8)
    if nib.shape[-1] % 2:
        nib = np.concatenate([nib, np.zeros(nib.shape[:-1] + (1,), np.uint8)], -1)
    return np.ascontiguousarray(nib[..., 0::2] | nib[..., 1::2] << 4)


class Cancelling:
    """A layer whose results are what an fp16 rounding of h = silu(..) * (..) takes away.

    Every gate is 32.  The up matrix gives outputs 2p and 2p + 1 the same value
    k (64 .. 127, exact in fp16), and 2p + 1 a little more: a part of 2^-16 to
    2^-13 of it, which 11 bits round off.  Down's codes of the two are d and -d,
    so that a row's results are the sums of d times these parts, all of one
    sign: without h's second part they are 0, or off by as much as they are.
    matrices: (planar codes, scales, values in 64 bits) by name."""

    def __init__(self, rng, qtype, down_type, count, hidden, ffn):
        assert hidden >= 64
        self.ffn = ffn
        pairs = ffn // 2
        lo, hi = (64, 128) if qtype == Q8_0 else (4, 8)  # codes; times `unit` they are 64 .. 127
        unit = np.float32(64 // lo)
        self.matrices = {}

        def add(name, codes, scales, kind):
            values = codes.astype(np.float64) * np.repeat(scales.astype(np.float64), R.BLOCK, -1)[..., :codes.shape[-1]]
            self.matrices[name] = (planar(codes, kind), scales, values)

        blocks = -(-hidden // R.BLOCK)
        gate = np.zeros((count, ffn, hidden), np.int8)
        gate[..., 0] = 4
        add("gate", gate, np.full((count, ffn, blocks), 8, np.float32), qtype)
        up, scales = np.zeros((count, ffn, hidden), np.int8), np.zeros((count, ffn, blocks), np.float32)
        scales[..., 0], scales[..., 1] = unit, unit * np.float32(2.0**-14)
        p = np.arange(pairs)
        up[:, 2 * p, 1] = up[:, 2 * p + 1, 1] = rng.integers(lo, hi, (count, pairs))
        up[:, 2 * p + 1, 32 + p % 32] = rng.integers(lo, hi, (count, pairs))
        add("up", up, scales, qtype)
        lo, hi = (64, 128) if down_type == Q8_0 else (4, 8)
        down = np.zeros((count, hidden, ffn), np.int8)
        down[..., 2 * p + 1] = rng.integers(lo, hi, (count, hidden, pairs))
        down[..., 2 * p] = -down[..., 2 * p + 1]
        scales = np.exp(rng.standard_normal((count, hidden, -(-ffn // R.BLOCK)))).astype(np.float32)
        add("down", down, scales, down_type)

    @staticmethod
    def rows(rng, tokens, hidden):
        """x: 1 and 1 for gates and k, then what the small parts are made of."""
        x = np.zeros((tokens, hidden), np.float32)
        x[:, :2] = 1
        x[:, 32:64] = rng.uniform(0.5, 1.0, (tokens, 32))
        return x

    def sums(self, ids, weights, x, parts=None):
        """Every token's sum and its bound; with parts (1 or 2) what an h of so many fp16 parts gives.

        Of an element of h: up to four roundings of k plus its small part, one of
        the product with silu's value, which both of a pair share up to its bits
        (8 units), and 2^-22 for the two parts.  Of the sums: the first parts
        are multiples of 16 (k 256 of a row whose largest is below 2^15), so that
        32 products with codes below 2^7 add up exactly, to 0; the second parts',
        64 additions of 2^-23, and those over blocks, experts and waves go by the
        result itself, since all of it has one sign."""
        tokens, top_k = ids.shape
        want, bound = np.zeros((2, tokens, x.shape[1]))
        x = x.astype(np.float64)
        steps = 64 + -(-self.ffn // R.BLOCK) + 4 * top_k + 16
        for e in range(len(self.matrices["gate"][2])):
            t, j = np.nonzero(ids == e)
            if not len(t):
                continue
            w = weights[t, j].astype(np.float64)[:, None]
            g, u = x[t] @ self.matrices["gate"][2][e].T, x[t] @ self.matrices["up"][2][e].T
            h = R.silu(g) * u
            if parts is not None:
                h = h.astype(np.float32).astype(np.float64)
                first = (h * 8).astype(np.float16)
                h = sum([first, (h * 8 - first).astype(np.float16)][:parts], np.zeros(h.shape)) / 8
            down = self.matrices["down"][2][e]
            y = h @ down.T
            np.add.at(want, t, w * y)
            np.add.at(bound, t, w * (h @ np.abs(down).T * 9 * 2.0**-24 + np.abs(y) * (8 * 2.0**-23 + steps * 2.0**-23)))
        return want, bound
