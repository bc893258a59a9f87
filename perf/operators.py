"""Performance cases of the paged 8-bit key/value cache: append, attention, read.

The cache of one transformer layer is a pool of pages.  A page holds
`page` positions of every key/value head as int8 codes, in blocks of 16
positions with one fp32 scale per block and head (for keys and for values):

  k       [page][kv head][block][dim / 16][16 positions][16 dims]    int8
  v       [page][kv head][block][dim / 16][16 dims][16 positions]    int8
  scales  [page][kv head][block][2]                                  fp32 (k, v)
  open    [slot][kv head][block parity][k, v][16][dim]               fp32

Three operators, over a ragged batch of sequences (sequence i brings count[i]
new tokens at positions start[i], start[i] + 1, ...):

  append     norms q and k per head (optional), rotates them by position,
             writes q back and quantizes k and v into the sequences' pages.
             A block that is not full is quantized as a whole from the fp32
             rows kept in `open`; the rows of a sequence's last two blocks
             are stored there.
  attention  causal attention of the new tokens over everything cached.
  read       the cached values of the tokens' positions as fp32 rows.

An append case is an append followed by the read of the blocks it wrote, so
that the values which the codes stand for are what comes back.

Head layouts are those of this library's synthetic models (9/3 and 14/2 heads
of 64) and generic ones; page tables are random permutations.
"""

import math
import os
import sys

import numpy as np
import torch

own = False

BLOCK = 16
EPS = 1e-6
THETA = 10000.0


def listed():
    return [
        # One user, one token into a block begun earlier; latency.
        _case("append_9x64_one", "append", 9, 3, 64, 64, 1, 37, 37, 1, 1),
        # 64 users decoding together, each at its own place.
        _case("append_14x64_64users", "append", 14, 2, 64, 64, 64, 16, 2040, 1, 1),
        # A prompt of 512 tokens.
        _case("append_14x64_prompt512", "append", 14, 2, 64, 64, 1, 0, 0, 512, 512),
        # Prompt chunks of eight users, with per-head norms; HBM.
        _case("append_32x128_norm_ragged", "append", 32, 8, 128, 32, 8, 0, 1800, 700, 2900, True),
        # The cached rows of one prompt read back (hand-over to an fp32 cache).
        _case("read_14x64_prompt500", "read", 14, 2, 64, 64, 1, 0, 0, 500, 500),
        # The same for eight long ragged sequences; HBM.
        _case("read_32x128_ragged", "read", 32, 8, 128, 64, 8, 0, 0, 2000, 8000),
        # One user's next token over a short history; latency.
        _case("attention_9x64_one_300", "attention", 9, 3, 64, 64, 1, 299, 299, 1, 1),
        # One user's next token over a long document: the history is split.
        _case("attention_14x64_one_32768", "attention", 14, 2, 64, 64, 1, 32767, 32767, 1, 1),
        # 64 users' next tokens over ragged histories; HBM.
        _case("attention_32x128_64users", "attention", 32, 8, 128, 64, 64, 120, 8191, 1, 1),
        # Drafted tokens checked together: a few rows per sequence.
        _case("attention_32x128_drafts", "attention", 32, 8, 128, 16, 16, 500, 3000, 3, 6),
        # A prompt of 512 tokens over itself.
        _case("attention_14x64_prompt512", "attention", 14, 2, 64, 64, 1, 0, 0, 512, 512),
        # A chunk of a long prompt over what came before; matrix cores.
        _case("attention_32x128_chunk2048", "attention", 32, 8, 128, 64, 1, 6144, 6144, 2048, 2048),
    ]


def _case(name, kind, heads, kv, dim, page, seqs, start_lo, start_hi, count_lo, count_hi, norm=False):
    c = {"kind": kind, "heads": heads, "kv": kv, "dim": dim, "page": page, "seqs": seqs, "start_lo": start_lo,
         "start_hi": start_hi, "count_lo": count_lo, "count_hi": count_hi, "norm": norm}
    return dict(c, name=name) if name else c


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    """One more case of the listed cases' ranges."""
    while True:
        kind = rng.choice(["append", "append", "read", "attention", "attention", "attention"])
        heads, kv, dim = rng.choice([(9, 3, 64), (14, 2, 64), (32, 8, 128), (12, 12, 64), (24, 3, 96), (8, 1, 256), (20, 4, 32)])
        page = rng.choice([16, 32, 48, 64, 128, 256])
        form = rng.choice(["tokens", "tokens", "drafts", "prompts", "chunks", "mixed"])
        norm = kind == "append" and rng.random() < 0.5
        if form == "tokens":
            a, b = sorted((_log(rng, 1, 16384), _log(rng, 1, 16384)))
            case = _case(None, kind, heads, kv, dim, page, _log(rng, 1, 64), a, b, 1, 1, norm)
        elif form == "drafts":
            a, b = sorted((_log(rng, 16, 8192), _log(rng, 16, 8192)))
            case = _case(None, kind, heads, kv, dim, page, _log(rng, 1, 32), a, b, 2, rng.randint(2, 9), norm)
        elif form == "prompts":
            a, b = sorted((_log(rng, 17, 3000), _log(rng, 17, 3000)))
            case = _case(None, kind, heads, kv, dim, page, rng.randint(1, 8), 0, 0, a, b, norm)
        elif form == "chunks":
            a, b = sorted((_log(rng, 16, 8192), _log(rng, 16, 8192)))
            case = _case(None, kind, heads, kv, dim, page, rng.randint(1, 6), a, b, 100, _log(rng, 101, 2048), norm)
        else:
            case = _case(None, kind, heads, kv, dim, page, rng.randint(2, 24), 0, _log(rng, 16, 4096), 1, _log(rng, 16, 1024), norm)
        tokens = sum(_counts(case))
        longest = max(s + c for s, c in zip(_starts(case), _counts(case)))
        # No dearer than the largest listed case, for the padded plain form too.
        volume = case["seqs"] * case["heads"] * max(_counts(case)) * longest
        reach = case["seqs"] * longest * case["kv"] * case["dim"]
        if kind != "attention" and tokens * (heads + 2 * kv) * dim > 14000 * 48 * 128:
            continue
        if kind == "attention" and (work(case)["flops"] > 2.2e11 or volume > 5.0e8 or reach > 5.0e8):
            continue
        return case


# ----------------------------------------------------- sequences and indexes


def _spread(lo, hi, i, phase):
    return lo + int((hi - lo + 1) * ((phase + 0.6180339887498949 * i) % 1.0))


def _starts(case):
    return [_spread(case["start_lo"], case["start_hi"], i, 0.37) for i in range(case["seqs"])]


def _counts(case):
    return [_spread(case["count_lo"], case["count_hi"], i, 0.83) for i in range(case["seqs"])]


def _inverse_frequencies(dim):
    return THETA ** (-torch.arange(0, dim, 2, dtype=torch.float64) / dim)


def _normal(gen, shape, std=1.0):
    return torch.empty(shape, dtype=torch.float32, device="cuda").normal_(0.0, std, generator=gen)


def _codes(gen, shape):
    """Codes of normal values in blocks of some hundred to some thousand: the largest of a block is 3 to 4 deviations."""
    x = torch.empty(shape, dtype=torch.float16, device="cuda").normal_(0.0, 34.0, generator=gen)
    return x.round_().clamp_(-127, 127).to(torch.int8)


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(int(seed))
    rs = np.random.RandomState(int(seed) % (1 << 31))
    heads, kv, dim, page, seqs = (case[k] for k in ("heads", "kv", "dim", "page", "seqs"))
    starts, counts = _starts(case), _counts(case)
    lens = [a + b for a, b in zip(starts, counts)]
    per = [-(-n // page) for n in lens]
    width, pages, tokens = max(per), sum(per) + 3, sum(counts)
    order = rs.permutation(pages)
    tables = np.zeros((seqs, width), dtype=np.int32)
    at = 0
    for i, n in enumerate(per):
        tables[i, :n] = order[at:at + n]
        at += n
    slots = rs.permutation(seqs).astype(np.int32)
    s = {"case": case, "slots": slots, "starts": np.array(starts, np.int32), "counts": np.array(counts, np.int32), "tables": tables, "pages": pages,
         "k": None, "v": None, "scales": None, "open": None}
    shape = (pages, kv, page // BLOCK, dim // 16, 16, 16)
    if case["kind"] == "append":
        s["k"] = torch.zeros(shape, dtype=torch.int8, device="cuda")
        s["v"] = torch.zeros(shape, dtype=torch.int8, device="cuda")
        s["scales"] = torch.zeros((pages, kv, page // BLOCK, 2), dtype=torch.float32, device="cuda")
        s["open"] = _normal(gen, (seqs, kv, 2, 2, BLOCK, dim))
        # One fused projection's rows: q, k and v of a token side by side.
        s["qkv"] = _normal(gen, (tokens, (heads + 2 * kv) * dim))
        s["q_out"] = torch.empty((tokens, heads * dim), dtype=torch.float32, device="cuda")
        s["wq"] = 1.0 + _normal(gen, (dim,), 0.1) if case["norm"] else None
        s["wk"] = 1.0 + _normal(gen, (dim,), 0.1) if case["norm"] else None
        angle = torch.arange(max(lens), dtype=torch.float64, device="cuda")[:, None] * _inverse_frequencies(dim).cuda()
        s["cos"], s["sin"] = angle.cos().float(), angle.sin().float()
    else:
        s["k"], s["v"] = _codes(gen, shape), _codes(gen, shape)
        s["scales"] = torch.exp(_normal(gen, (pages, kv, page // BLOCK, 2), 0.2)) / 34.0
        s["open"] = torch.zeros((seqs, kv, 2, 2, BLOCK, dim), dtype=torch.float32, device="cuda")
        s["q"] = _normal(gen, (tokens, heads * dim))
        s["out"] = torch.empty((tokens, heads * dim), dtype=torch.float32, device="cuda")
    # Read: every new token's row, for an append from the first row of the first block that it writes.
    r_starts = [(a // BLOCK) * BLOCK if case["kind"] == "append" else a for a in starts]
    r_counts = [n - a for a, n in zip(r_starts, lens)]
    s["read_k"] = torch.empty((sum(r_counts), kv * dim), dtype=torch.float32, device="cuda")
    s["read_v"] = torch.empty((sum(r_counts), kv * dim), dtype=torch.float32, device="cuda")
    s.update(_indexes(case, s, r_starts, r_counts))
    if own:
        _own_prepare(case, s, np.array(r_starts, np.int32), np.array(r_counts, np.int32))
    return s


def _ragged(starts, counts):
    """(sequence, position) of every row of a ragged batch."""
    seq = np.repeat(np.arange(len(counts)), counts)
    first = np.cumsum(counts) - np.asarray(counts)
    return seq, np.asarray(starts)[seq] + np.arange(len(seq)) - first[seq]


def _indexes(case, s, r_starts, r_counts):
    """The plain form's plan: where each row comes from and goes to."""
    page, tables = case["page"], s["tables"]
    starts, counts = s["starts"], s["counts"]
    seq, pos = _ragged(starts, counts)
    d = {"seq": seq, "pos": pos, "tok": pos - starts[seq]}
    rseq, rpos = _ragged(r_starts, r_counts)
    d["r_page"], d["r_block"], d["r_row"] = tables[rseq, rpos // page], rpos % page // BLOCK, rpos % BLOCK
    if case["kind"] == "append":
        lens = starts + counts
        first, last = starts // BLOCK, (lens - 1) // BLOCK
        bseq, bidx = _ragged(first, last - first + 1)
        at = bidx[:, None] * BLOCK + np.arange(BLOCK)  # position of each row of each block
        row0 = (np.cumsum(counts) - counts)[bseq]
        new = (at >= starts[bseq][:, None]) & (at < lens[bseq][:, None])
        old = at < starts[bseq][:, None]
        d["b_new"] = np.where(new, row0[:, None] + at - starts[bseq][:, None], 0)
        d["b_is_new"], d["b_is_old"] = new, old
        d["b_slot"], d["b_parity"] = s["slots"][bseq], bidx % 2
        d["b_page"], d["b_block"] = tables[bseq, bidx * BLOCK // page], bidx * BLOCK % page // BLOCK
        keep = np.nonzero(pos // BLOCK >= last[seq] - 1)[0]  # rows of the last two blocks stay in `open`
        d["o_tok"], d["o_slot"] = keep, s["slots"][seq[keep]]
        d["o_parity"], d["o_row"] = pos[keep] // BLOCK % 2, pos[keep] % BLOCK
    if case["kind"] == "attention":
        width = tables.shape[1]
        d["tables"] = tables.astype(np.int64)
        d["limit"] = np.array(starts)[:, None] + np.arange(int(counts.max()))  # the row's own position
        d["cols"] = np.arange(width * page)
    return {"x_" + k: torch.from_numpy(np.ascontiguousarray(v)).cuda() for k, v in d.items()}


def _own_prepare(case, s, r_starts, r_counts):
    sys.path.insert(0, os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "llm-inference-cpp_amd"))
    import llmi_hip as H

    H.init(0)
    torch.cuda.synchronize()
    shape = H.Kv8Shape(heads=case["heads"], kv_heads=case["kv"], head_dim=case["dim"], page_tokens=case["page"], pages=s["pages"], slots=case["seqs"])
    s["layer"] = H.Kv8Layer(s["k"].data_ptr(), s["v"].data_ptr(), s["scales"].data_ptr(), s["open"].data_ptr())
    s["plan"] = H.Kv8Plan(shape, case["seqs"], int(s["counts"].sum()))
    s["plan"].set(s["slots"], s["starts"], s["counts"], s["tables"])
    if case["kind"] == "append":
        s["read_plan"] = H.Kv8Plan(shape, case["seqs"], int(r_counts.sum()))
        s["read_plan"].set(s["slots"], r_starts, r_counts, s["tables"])


# --------------------------------------------------------------------- run


def run(s):
    return {"append": _append, "read": _read, "attention": _attention}[s["case"]["kind"]](s)


def _append(s):
    case = s["case"]
    heads, kv, dim = case["heads"], case["kv"], case["dim"]
    if own:
        row = (heads + 2 * kv) * dim
        q = s["qkv"].data_ptr()
        k, v = q + 4 * heads * dim, q + 4 * (heads + kv) * dim
        s["plan"].append(s["layer"], q, k, v, s["q_out"].data_ptr(), q_stride=row, k_stride=row, v_stride=row,
                         q_norm=s["wq"].data_ptr() if case["norm"] else None, k_norm=s["wk"].data_ptr() if case["norm"] else None, eps=EPS,
                         cos=s["cos"].data_ptr(), sin=s["sin"].data_ptr(), positions=s["cos"].shape[0])
        s["read_plan"].read(s["layer"], s["read_k"].data_ptr(), s["read_v"].data_ptr())
        return {"q": s["q_out"], "k": s["read_k"], "v": s["read_v"], "open": s["open"]}
    # 64 bits up to the one rounding to fp32: the codes sit next to borders.
    qkv = s["qkv"].double()
    q = qkv[:, : heads * dim].unflatten(1, (heads, dim))
    k = qkv[:, heads * dim : (heads + kv) * dim].unflatten(1, (kv, dim))
    v = s["qkv"][:, (heads + kv) * dim :].unflatten(1, (kv, dim))
    if case["norm"]:
        q = q / (q.square().mean(-1, keepdim=True) + EPS).sqrt() * s["wq"].double()
        k = k / (k.square().mean(-1, keepdim=True) + EPS).sqrt() * s["wk"].double()
    c, n = s["cos"][s["x_pos"]].double()[:, None], s["sin"][s["x_pos"]].double()[:, None]
    q, k = _rotate(q, c, n).float(), _rotate(k, c, n).float()
    kv_new = torch.stack([k, v], 2)  # [token][kv head][2][dim]
    new, old = s["x_b_is_new"][:, None, None, :, None], s["x_b_is_old"][:, None, None, :, None]
    held = s["open"][s["x_b_slot"], :, s["x_b_parity"]]  # [block][kv head][2][16][dim]
    rows = torch.where(new, kv_new[s["x_b_new"]].permute(0, 2, 3, 1, 4), torch.where(old, held, torch.zeros_like(held)))
    scale = (rows.abs().amax((3, 4)).double() / 127).float()
    codes = (rows.double() / torch.where(scale > 0, scale, torch.ones_like(scale)).double()[..., None, None]).round().clamp(-127, 127).to(torch.int8)
    codes = codes.unflatten(4, (dim // 16, 16))  # [block][kv head][2][16 positions][dim / 16][16]
    s["k"][s["x_b_page"], :, s["x_b_block"]] = codes[:, :, 0].permute(0, 1, 3, 2, 4)
    s["v"][s["x_b_page"], :, s["x_b_block"]] = codes[:, :, 1].permute(0, 1, 3, 4, 2)
    s["scales"][s["x_b_page"], :, s["x_b_block"]] = scale
    s["open"][s["x_o_slot"], :, s["x_o_parity"], :, s["x_o_row"]] = kv_new[s["x_o_tok"]]
    return {"q": q.flatten(1), "open": s["open"], **_read(s)}


def _rotate(x, c, n):
    a, b = x.chunk(2, -1)
    return torch.cat([a * c - b * n, b * c + a * n], -1)


def _read(s):
    if own:
        s["plan"].read(s["layer"], s["read_k"].data_ptr(), s["read_v"].data_ptr())
        return {"k": s["read_k"], "v": s["read_v"]}
    scale = s["scales"][s["x_r_page"], :, s["x_r_block"]]  # [row][kv head][2]
    k = s["k"][s["x_r_page"], :, s["x_r_block"], :, s["x_r_row"]]  # [row][kv head][dim / 16][16]
    v = s["v"][s["x_r_page"], :, s["x_r_block"], :, :, s["x_r_row"]]
    return {"k": (k.flatten(2).float() * scale[..., :1]).flatten(1), "v": (v.flatten(2).float() * scale[..., 1:]).flatten(1)}


def _attention(s):
    case = s["case"]
    heads, kv, dim = case["heads"], case["kv"], case["dim"]
    if own:
        s["plan"].attention(s["layer"], s["q"].data_ptr(), dim ** -0.5, s["out"].data_ptr())
        return s["out"]
    group, most = heads // kv, s["x_limit"].shape[1]
    tables = s["x_tables"]
    scale = s["scales"][tables].permute(0, 2, 1, 3, 4).flatten(2, 3)  # [sequence][kv head][block][2]
    # [sequence][page][kv head][block][dim / 16][position][dim] -> [sequence][kv head][position][dim]
    k = s["k"][tables].permute(0, 2, 1, 3, 5, 4, 6).flatten(5).flatten(2, 3).float() * scale[..., 0, None, None]
    v = s["v"][tables].permute(0, 2, 1, 3, 6, 4, 5).flatten(5).flatten(2, 3).float() * scale[..., 1, None, None]
    k, v = k.flatten(2, 3), v.flatten(2, 3)
    q = torch.zeros((case["seqs"], most, kv, group, dim), dtype=torch.float32, device="cuda")
    q[s["x_seq"], s["x_tok"]] = s["q"].unflatten(1, (kv, group, dim))
    q = q.permute(0, 2, 1, 3, 4).flatten(2, 3)  # [sequence][kv head][token, group][dim]
    p = torch.matmul(q, k.transpose(2, 3).contiguous()).mul_(dim ** -0.5).unflatten(2, (most, group))
    p.masked_fill_((s["x_cols"] > s["x_limit"][..., None])[:, None, :, None], float("-inf"))
    p.sub_(p.amax(-1, keepdim=True)).exp_()
    total = p.sum(-1, keepdim=True)
    o = torch.matmul(p.flatten(2, 3), v).unflatten(2, (most, group)) / total
    return o.permute(0, 2, 1, 3, 4)[s["x_seq"], s["x_tok"]].flatten(1)


# -------------------------------------------------------------------- work


def work(case):
    heads, kv, dim = case["heads"], case["kv"], case["dim"]
    starts, counts = _starts(case), _counts(case)
    tokens = sum(counts)
    blocks = lambda lo, hi: -(-hi // BLOCK) - lo // BLOCK  # noqa: E731
    if case["kind"] == "read":
        held = sum(blocks(a, a + n) for a, n in zip(starts, counts))
        return {"bytes": tokens * kv * dim * (2 + 8) + held * kv * 8, "flops": 2 * tokens * kv * dim}
    if case["kind"] == "append":
        held = sum(blocks(a, a + n) for a, n in zip(starts, counts))
        back = sum(a % BLOCK for a in starts)  # rows of begun blocks, read from `open`
        rows = tokens + back                   # rows quantized, and read again as values
        kept = sum(min(n, a + n - max(0, ((a + n - 1) // BLOCK - 1) * BLOCK)) for a, n in zip(starts, counts))
        moved = tokens * (heads + 2 * kv) * dim * 4 + tokens * heads * dim * 4 + tokens * dim * 4  # q, k, v in; q out; cos, sin
        moved += 8 * back * kv * dim + 8 * kept * kv * dim + 2 * rows * kv * dim + 8 * held * kv   # open rows; codes, scales
        moved += rows * kv * dim * (2 + 8) + held * kv * 8                                         # the read
        return {"bytes": moved, "flops": tokens * (heads + kv) * dim * (10 if case["norm"] else 6) + rows * kv * dim * 8}
    seen = sum(n * a + n * (n + 1) // 2 for a, n in zip(starts, counts))
    length = sum(a + n for a, n in zip(starts, counts))
    held = sum(blocks(0, a + n) for a, n in zip(starts, counts))
    return {"bytes": length * kv * dim * 2 + held * kv * 8 + 2 * tokens * heads * dim * 4, "flops": 4 * dim * heads * seen}


# ------------------------------------------------------------------- exact


def exact(case, seed):
    s = prepare(case, seed)
    return {"append": _exact_append, "read": _exact_read, "attention": _exact_attention}[case["kind"]](case, s)


def _page_values(case, s, i, upto):
    """Keys and values of sequence i's first `upto` positions, [position][kv head][dim], in 64 bits."""
    kv, dim, page = case["kv"], case["dim"], case["page"]
    ids = torch.from_numpy(s["tables"][i][: -(-upto // page)].astype(np.int64)).cuda()
    sc = s["scales"][ids].double()
    k = s["k"][ids].double() * sc[..., 0][..., None, None, None]
    v = s["v"][ids].double() * sc[..., 1][..., None, None, None]
    k = torch.einsum("phbgtd->pbthgd", k).reshape(-1, kv, dim)
    v = torch.einsum("phbgdt->pbthgd", v).reshape(-1, kv, dim)
    return k[:upto], v[:upto]


def _exact_read(case, s):
    ks, vs = [], []
    for i, (a, n) in enumerate(zip(s["starts"], s["counts"])):
        k, v = _page_values(case, s, i, int(a + n))
        ks.append(k[int(a):].flatten(1))
        vs.append(v[int(a):].flatten(1))
    return {"k": torch.cat(ks), "v": torch.cat(vs)}


def _exact_append(case, s):
    heads, kv, dim = case["heads"], case["kv"], case["dim"]
    x = s["qkv"].double()
    turned = []
    for part, w in ((x[:, : heads * dim], s["wq"]), (x[:, heads * dim : (heads + kv) * dim], s["wk"])):
        part = part.reshape(len(x), -1, dim)
        if w is not None:
            part = part * w.double() * torch.rsqrt((part * part).sum(-1, keepdim=True) / dim + EPS)
        z = torch.complex(part[..., : dim // 2], part[..., dim // 2 :])
        z = z * torch.complex(s["cos"].double(), s["sin"].double())[s["x_pos"]][:, None]
        turned.append(torch.cat([z.real, z.imag], -1))
    q, k = turned
    v = x[:, (heads + kv) * dim :].reshape(len(x), kv, dim)
    opened = s["open"].double()
    ks, vs, row = [], [], 0
    for a, n, slot in zip(s["starts"].tolist(), s["counts"].tolist(), s["slots"].tolist()):
        a0, end = a // BLOCK * BLOCK, a + n
        for out, new, which in ((ks, k, 0), (vs, v, 1)):
            held = s["open"][slot, :, a0 // BLOCK % 2, which, : a - a0].double().transpose(0, 1)
            # The cache takes values rounded to 32 bits.
            rows = torch.cat([held, new[row : row + n].float().double()])
            pad = torch.zeros((-len(rows) % BLOCK, kv, dim), dtype=torch.float64, device="cuda")
            blocks = torch.cat([rows, pad]).reshape(-1, BLOCK, kv, dim)
            step = (blocks.abs().amax((1, 3), keepdim=True) / 127).float().double()
            whole = torch.where(step > 0, (blocks / step).round(), 0.0).clamp(-127, 127)
            out.append((whole * step).reshape(-1, kv, dim)[: len(rows)].flatten(1))
            last = (end - 1) // BLOCK
            for b in range(max(a0 // BLOCK, last - 1), last + 1):
                lo, hi = max(a, b * BLOCK), min(end, (b + 1) * BLOCK)
                opened[slot, :, b % 2, which, lo - b * BLOCK : hi - b * BLOCK] = new[row + lo - a : row + hi - a].transpose(0, 1)
        row += n
    return {"q": q.flatten(1), "k": torch.cat(ks), "v": torch.cat(vs), "open": opened}


def _exact_attention(case, s):
    heads, kv, dim = case["heads"], case["kv"], case["dim"]
    outs, row = [], 0
    for i, (a, n) in enumerate(zip(s["starts"].tolist(), s["counts"].tolist())):
        k, v = _page_values(case, s, i, a + n)
        q = s["q"][row : row + n].double().reshape(n, kv, heads // kv, dim)
        hidden = torch.arange(a + n, device="cuda") > torch.arange(a, a + n, device="cuda")[:, None]
        o = torch.empty((n, kv, heads // kv, dim), dtype=torch.float64, device="cuda")
        for h in range(kv):
            score = torch.tensordot(q[:, h], k[:, h], ([2], [1])) / math.sqrt(dim)  # [token][group][position]
            score = score.masked_fill(hidden[:, None], float("-inf"))
            o[:, h] = torch.tensordot(torch.softmax(score, -1), v[:, h], ([2], [0]))
        outs.append(o.reshape(n, heads * dim))
        row += n
    return torch.cat(outs)
