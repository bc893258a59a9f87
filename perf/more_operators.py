"""Performance cases of a layer of experts: router, grouped products, expert MLPs.

The experts' matrices hold quantized weights as the library's other products do
(planar layout of one expert after the other):

  codes   [expert][out][in]            int8 (q8_0)
          [expert][out][ceil(in / 2)]  bytes of two 4-bit codes + 8, the even element low (q4_0)
  scales  [expert][out][ceil(in / 32)] fp32, one of every 32 weights

Three operators, over tokens that each choose top_k experts:

  route   the top_k largest logits of every token and their softmax weights.
          Logits of -inf (experts that are switched off) are never chosen: where
          fewer are left, ids are -1 and weights 0.
  matmul  y[slot] = W[ids[slot]] x[slot / top_k]; slots with id -1 (padding
          tokens) keep what y held.
  mlp     y[t] = residual[t] + sum over j of weights[t][j] *
          down(silu(gate x[t]) * up x[t]), the matrices of expert ids[t][j].

Sizes are those of this library's synthetic models (576 / 1536 and 896 / 4864)
and generic ones.  Experts are chosen as trained routers do: some are several
times as popular as others.
"""

import math
import os
import sys

import numpy as np
import torch

own = False

BLOCK = 32
BITS = {"q8_0": 8, "q4_0": 4}


def listed():
    return [
        # One token of a decoding user: latency.
        _route("route_64_one", 1, 64, 8, 0.0, True),
        # A batch of decoding users, few experts.
        _route("route_8_64users", 64, 8, 2, 0.0, True),
        # Long prompts; a tenth of the experts switched off, weights not renormalised.
        _route("route_128_tokens8192", 8192, 128, 8, 0.1, False),
        # One token's two experts, the smallest matrices: latency.
        _matmul("matmul_q4_576x1536_one", "q4_0", 1, 8, 2, 576, 1536),
        # 64 users decoding: nearly every expert, a few rows each; HBM.
        _matmul("matmul_q8_2048x1024_64users", "q8_0", 64, 64, 8, 2048, 1024),
        # Ragged sizes, padding tokens.
        _matmul("matmul_q8_1000x777_odd", "q8_0", 333, 13, 3, 1000, 777, pad=0.1),
        # A prompt through wide experts; matrix cores.
        _matmul("matmul_q4_896x4864_prompt2048", "q4_0", 2048, 16, 2, 896, 4864),
        # One token's layer, eight small experts of 64.
        _mlp("mlp_q4_2048x1024_one", "q4_0", "q4_0", 1, 64, 8, 2048, 1024),
        # One token's layer, two large experts of eight; HBM.
        _mlp("mlp_q8_4096x8192_one", "q8_0", "q8_0", 1, 8, 2, 4096, 8192, residual=True),
        # 64 users' layer; HBM.
        _mlp("mlp_q4_2048x1024_64users", "q4_0", "q4_0", 64, 64, 8, 2048, 1024, residual=True),
        # A prompt of 512 tokens.
        _mlp("mlp_q8_896x4864_prompt512", "q8_0", "q8_0", 512, 8, 2, 896, 4864),
        # A long prompt over many experts; matrix cores.
        _mlp("mlp_q4_2048x1024_prompt4096", "q4_0", "q4_0", 4096, 64, 8, 2048, 1024, residual=True),
    ]


def _named(name, **case):
    return dict(case, name=name) if name else case


def _route(name, tokens, experts, top_k, off, renormalise):
    return _named(name, kind="route", tokens=tokens, experts=experts, top_k=top_k, off=off, renormalise=renormalise)


def _matmul(name, type, tokens, experts, top_k, hidden, ffn, pad=0.0):
    return _named(name, kind="matmul", type=type, down=type, tokens=tokens, experts=experts, top_k=top_k, hidden=hidden,
                  ffn=ffn, pad=pad, residual=False)


def _mlp(name, type, down, tokens, experts, top_k, hidden, ffn, pad=0.0, residual=False):
    return _named(name, kind="mlp", type=type, down=down, tokens=tokens, experts=experts, top_k=top_k, hidden=hidden,
                  ffn=ffn, pad=pad, residual=residual)


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    """One more case of the listed cases' ranges."""
    while True:
        kind = rng.choice(["route", "matmul", "matmul", "mlp", "mlp", "mlp"])
        experts = rng.choice([4, 8, 8, 13, 16, 32, 60, 64, 128])
        top_k = rng.choice([k for k in (1, 2, 2, 3, 4, 6, 8) if k <= experts])
        if kind == "route":
            return _route(None, _log(rng, 1, 8192), experts, top_k, rng.choice([0.0, 0.0, 0.1, 0.5]), rng.random() < 0.5)
        hidden, ffn = _log(rng, 256, 4096), _log(rng, 256, 8192)
        # Most models have multiples of 64; others have to work too.
        if rng.random() < 0.7:
            hidden, ffn = -(-hidden // 64) * 64, -(-ffn // 64) * 64
        form = rng.choice(["one", "few", "users", "prompt", "prompt"])
        tokens = {"one": 1, "few": rng.randint(2, 9), "users": _log(rng, 10, 256), "prompt": _log(rng, 128, 4096)}[form]
        type = rng.choice(["q4_0", "q8_0"])
        pad = rng.choice([0.0, 0.0, 0.05, 0.3]) if tokens > 1 else 0.0
        if kind == "matmul":
            case = _matmul(None, type, tokens, experts, top_k, hidden, ffn, pad)
        else:
            case = _mlp(None, type, rng.choice([type, type, "q8_0"]), tokens, experts, top_k, hidden, ffn, pad, rng.random() < 0.5)
        # No dearer than the largest listed cases, in products, weights held and results.
        mats = 1 if kind == "matmul" else 3
        if 2 * mats * tokens * top_k * hidden * ffn > 4.1e11 or mats * experts * hidden * ffn > 8.0e8 or tokens * top_k * max(hidden, ffn) > 7.0e7:
            continue
        return case


# ------------------------------------------------------------------ inputs


def _normal(gen, shape, std=1.0):
    return torch.empty(shape, dtype=torch.float32, device="cuda").normal_(0.0, std, generator=gen)


def _matrices(gen, type, experts, out, inner):
    """Random experts as quantized normal weights have them, results of size 1."""
    blocks = -(-inner // BLOCK)
    scales = torch.exp(_normal(gen, (experts, out, blocks), 0.25)) / math.sqrt(inner)
    codes = torch.empty((experts, out, inner), dtype=torch.int8, device="cuda")
    spread, top = (42.0, 127) if type == "q8_0" else (3.0, 7)
    for e in range(experts):
        codes[e] = _normal(gen, (out, inner), spread).round_().clamp_(-top - (type == "q4_0"), top).to(torch.int8)
    if type == "q4_0":
        even, odd = codes[..., 0::2] + 8, codes[..., 1::2] + 8
        if inner % 2:  # the last byte's high half is not used
            odd = torch.nn.functional.pad(odd, (0, 1))
        codes = (even | (odd << 4)).view(torch.uint8)
    return {"type": type, "experts": experts, "out": out, "in": inner, "codes": codes.contiguous(), "scales": scales / spread}


def _logits(gen, tokens, experts):
    """A router's logits: some experts are more popular than others."""
    return _normal(gen, (tokens, experts)) * 1.5 + _normal(gen, (experts,), 0.7)


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(int(seed))
    tokens, experts, top_k = case["tokens"], case["experts"], case["top_k"]
    s = {"case": case}
    logits = _logits(gen, tokens, experts)
    if case["kind"] == "route":
        off = torch.empty((tokens, experts), device="cuda").uniform_(generator=gen) < case["off"]
        s["logits"] = logits.masked_fill_(off, float("-inf"))
        s["ids"] = torch.empty((tokens, top_k), dtype=torch.int32, device="cuda")
        s["weights"] = torch.empty((tokens, top_k), dtype=torch.float32, device="cuda")
    else:
        hidden, ffn = case["hidden"], case["ffn"]
        top, ids = logits.sort(dim=1, descending=True, stable=True)
        s["ids"] = ids[:, :top_k].to(torch.int32).contiguous()
        s["weights"] = torch.exp(top[:, :top_k] - top[:, :1])
        s["weights"] /= s["weights"].sum(1, keepdim=True)
        s["ids"][torch.empty(tokens, device="cuda").uniform_(generator=gen) < case["pad"]] = -1
        # A few channels of the hidden state are much larger than the others.
        loud = torch.exp(_normal(gen, (hidden,), 0.3)) * (1.0 + 15.0 * (torch.arange(hidden, device="cuda") % 301 == 7))
        s["x"] = _normal(gen, (tokens, hidden)) * loud
        s["gate"] = _matrices(gen, case["type"], experts, ffn, hidden)
        width = ffn if case["kind"] == "matmul" else hidden
        rows = tokens * top_k if case["kind"] == "matmul" else tokens
        s["y"] = torch.zeros((rows, width), dtype=torch.float32, device="cuda")
        s["residual"] = _normal(gen, (tokens, hidden)) if case["residual"] else None
        if case["kind"] == "mlp":
            s["up"] = _matrices(gen, case["type"], experts, ffn, hidden)
            s["down"] = _matrices(gen, case["down"], experts, hidden, ffn)
    if own:
        _own_prepare(case, s)
    return s


def _own_prepare(case, s):
    sys.path.insert(0, os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "llm-inference-cpp_amd"))
    import llmi_hip as H

    H.init(0)
    torch.cuda.synchronize()
    s["H"] = H
    if case["kind"] == "route":
        return
    for name in ("gate", "up", "down"):
        if name in s:
            m = s[name]
            s["h_" + name] = H.Experts.upload_dev(m["codes"].data_ptr(), m["scales"].data_ptr(), m["experts"], m["out"], m["in"],
                                                  H.Q8_0 if m["type"] == "q8_0" else H.Q4_0)
    if case["kind"] == "matmul":
        size = H.moe_matmul_bytes(s["h_gate"], case["tokens"] * case["top_k"], case["top_k"])
    else:
        size = H.moe_mlp_bytes(s["h_gate"], s["h_down"], case["tokens"], case["top_k"])
    s["work"] = torch.empty(max(size, 1), dtype=torch.uint8, device="cuda")


# --------------------------------------------------------------------- run


def run(s):
    return {"route": _run_route, "matmul": _run_matmul, "mlp": _run_mlp}[s["case"]["kind"]](s)


def _run_route(s):
    case = s["case"]
    if own:
        s["H"].moe_route(s["logits"].data_ptr(), case["tokens"], case["experts"], case["top_k"], s["ids"].data_ptr(),
                         s["weights"].data_ptr(), renormalise=case["renormalise"])
        return {"ids": s["ids"], "weights": s["weights"]}
    top, ids = s["logits"].sort(dim=1, descending=True, stable=True)
    p = torch.exp(top - top[:, :1].clamp_min(torch.finfo(torch.float32).min))  # all switched off: 0
    total = p[:, : case["top_k"]].sum(1, keepdim=True) if case["renormalise"] else p.sum(1, keepdim=True)
    p, top, ids = p[:, : case["top_k"]], top[:, : case["top_k"]], ids[:, : case["top_k"]]
    return {"ids": torch.where(top > float("-inf"), ids, -1).to(torch.int32), "weights": torch.where(p > 0, p / total, p)}


def _dense(m, e):
    """Expert e's matrix in fp32."""
    codes = m["codes"][e]
    if m["type"] == "q4_0":
        codes = torch.stack([codes & 15, codes >> 4], -1).flatten(1)[:, : m["in"]].float() - 8.0
    else:
        codes = codes.float()
    return codes * m["scales"][e].repeat_interleave(BLOCK, 1)[:, : m["in"]]


def _groups(ids, experts):
    """The slots of every expert that has any."""
    order = torch.sort(ids.flatten(), dim=0, stable=True)[1]
    counts = torch.bincount(ids.flatten() + 1, minlength=experts + 1).tolist()  # a dense program needs them on the host
    at = counts[0]
    for e in range(experts):
        n = counts[e + 1]
        if n:
            yield e, order[at : at + n]
        at += n


def _run_matmul(s):
    case = s["case"]
    if own:
        s["H"].moe_matmul(s["h_gate"], s["ids"].data_ptr(), case["tokens"] * case["top_k"], s["x"].data_ptr(), s["y"].data_ptr(),
                          s["work"].data_ptr(), s["work"].numel(), per_row=case["top_k"])
        return s["y"]
    for e, slots in _groups(s["ids"], case["experts"]):
        s["y"][slots] = torch.mm(s["x"][slots // case["top_k"]], _dense(s["gate"], e).t())
    return s["y"]


def _run_mlp(s):
    case = s["case"]
    if own:
        s["H"].moe_mlp(s["h_gate"], s["h_up"], s["h_down"], s["ids"].data_ptr(), s["weights"].data_ptr(), case["tokens"],
                       case["top_k"], s["x"].data_ptr(), s["y"].data_ptr(), s["work"].data_ptr(), s["work"].numel(),
                       residual=None if s["residual"] is None else s["residual"].data_ptr())
        return s["y"]
    y = torch.zeros_like(s["y"]) if s["residual"] is None else s["residual"].clone()
    weights = s["weights"].flatten()
    for e, slots in _groups(s["ids"], case["experts"]):
        rows = slots // case["top_k"]
        x = s["x"][rows]
        g = torch.mm(x, _dense(s["gate"], e).t())
        h = g / (1.0 + torch.exp(-g)) * torch.mm(x, _dense(s["up"], e).t())
        y.index_add_(0, rows, weights[slots, None] * torch.mm(h, _dense(s["down"], e).t()))
    return y


# -------------------------------------------------------------------- work


def _touched(case):
    """About how many experts have any token, and how many slots are not padding."""
    if case["tokens"] == 1:
        return case["top_k"], case["top_k"]
    rs = np.random.RandomState(1)
    logits = rs.standard_normal((case["tokens"], case["experts"])) * 1.5 + 0.7 * rs.standard_normal(case["experts"])
    ids = np.argsort(-logits, 1)[rs.uniform(size=case["tokens"]) >= case["pad"], : case["top_k"]]
    return len(np.unique(ids)), ids.size


def work(case):
    tokens, experts, top_k = case["tokens"], case["experts"], case["top_k"]
    if case["kind"] == "route":
        return {"bytes": 4 * tokens * experts + 8 * tokens * top_k, "flops": 3 * tokens * experts}
    hidden, ffn = case["hidden"], case["ffn"]
    touched, slots = _touched(case)

    def held(type, out, inner):
        return touched * out * ((inner * BITS[type] + 7) // 8 + 4 * -(-inner // BLOCK))

    if case["kind"] == "matmul":
        return {"bytes": held(case["type"], ffn, hidden) + 4 * tokens * (hidden + top_k) + 4 * slots * ffn, "flops": 2 * slots * hidden * ffn}
    rows = tokens * hidden * 4 * (3 if case["residual"] else 2)
    return {"bytes": 2 * held(case["type"], ffn, hidden) + held(case["down"], hidden, ffn) + rows + 8 * tokens * top_k,
            "flops": 6 * slots * hidden * ffn}


# ------------------------------------------------------------------- exact


def exact(case, seed):
    s = prepare(case, seed)
    if case["kind"] == "route":
        return _exact_route(case, s)
    top_k, x = case["top_k"], s["x"].double()
    ids = s["ids"].long()
    slots = torch.zeros((case["tokens"], top_k, s["y"].shape[1]), dtype=torch.float64, device="cuda")
    for e in range(case["experts"]):
        t, j = torch.nonzero(ids == e, as_tuple=True)
        if not len(t):
            continue
        r = x[t] @ _exact_matrix(s["gate"], e)
        if case["kind"] == "mlp":
            r = r * torch.sigmoid(r) * (x[t] @ _exact_matrix(s["up"], e))
            r = r @ _exact_matrix(s["down"], e)
        slots[t, j] = r
    if case["kind"] == "matmul":
        return slots.flatten(0, 1)
    total = (slots * s["weights"].double()[..., None]).sum(1)
    return total if s["residual"] is None else total + s["residual"].double()


def _exact_matrix(m, e):
    """Expert e's matrix, transposed, in 64 bits."""
    w = torch.zeros((m["in"], m["out"]), dtype=torch.float64, device="cuda")
    codes = m["codes"][e].t()
    if m["type"] == "q8_0":
        w += codes
    else:
        w[0::2] = (codes % 16).double() - 8
        w[1::2] = (codes[: m["in"] // 2] // 16).double() - 8
    for b in range(m["scales"].shape[2]):
        w[b * BLOCK : (b + 1) * BLOCK] *= m["scales"][e, :, b].double()
    return w


def _exact_route(case, s):
    left = s["logits"].double()
    top = left.amax(1, keepdim=True)
    top = torch.where(torch.isinf(top), 0.0, top)
    whole = torch.exp(left - top).sum(1)
    ids, weights = [], []
    index = torch.arange(case["experts"], device="cuda")
    for _ in range(case["top_k"]):
        best = left.amax(1, keepdim=True)
        first = torch.where(left == best, index, case["experts"]).amin(1)
        live = best[:, 0] > float("-inf")
        ids.append(torch.where(live, first, -1))
        weights.append(torch.where(live, torch.exp(best - top)[:, 0], 0.0))
        left = torch.where(index == first[:, None], float("-inf"), left)
    weights = torch.stack(weights, 1)
    total = weights.sum(1) if case["renormalise"] else whole
    return {"ids": torch.stack(ids, 1).to(torch.int32), "weights": weights / torch.where(total > 0, total, 1.0)[:, None]}
