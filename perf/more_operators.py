"""What a step reads, in 8 bits: operators for weights and for the cache of keys and values, as cases that can be timed and checked one by one.

* ``kind: "product"``  x W^T for a weight of 8-bit floating point numbers (e4m3) with a scale for each block of 128 x 128; the rows of x are brought to 8 bits
  within the call, with a scale for each row and 128 columns.
* ``kind: "append"``   the heads of a projection: norm and rotation of queries and keys, and the write of keys and values into pages of 64 tokens
  held in 8 bits, with a scale (a power of two) for each page and head.
* ``kind: "decode"``   one query token for each sequence over such a cache.
* ``kind: "prompt"``   the queries of prompts, or of their later pieces, over such a cache, causal.

Lengths within a case follow from its ``layout`` number, so that a case says all of its sizes; the seed gives the numbers.
"""
from __future__ import annotations

import math
import random

import torch

own = False

PAGE = 64                     # tokens a page, and a block of the cache's scales
GROUP = 128                   # columns (and rows of a weight) that share a scale
TOP = 448.0                   # the largest e4m3 number
EPS = 1e-6                    # of the norms
E4M3 = torch.float8_e4m3fn
TYPES = {"bf16": torch.bfloat16, "fp32": torch.float32}


# ----------------------------------------------------------------------------- cases
def listed() -> list[dict]:
    def product(name, rows, features, inputs, dtype="bf16"):
        return {"name": name, "kind": "product", "rows": rows, "features": features, "inputs": inputs, "dtype": dtype}

    def cached(name, kind, batch, tokens, past, heads, kv_heads, dim, dtype="bf16", layout=0):
        return {"name": name, "kind": kind, "batch": batch, "tokens": tokens, "past": past, "heads": heads, "kv_heads": kv_heads,
                "head_dim": dim, "dtype": dtype, "layout": layout}

    return [
        # one user's next token: the output projection of the 0.6B shape, where latency counts
        product("one-token", 1, 1024, 2048),
        # eight users: the down projection of the 8B shape, bound by reading the weight
        product("down-8", 8, 4096, 12288),
        # a short prompt of odd length: the output projection of the 32B shape
        product("prompt-333", 333, 5120, 8192),
        # the 32-bit path, with sizes that end inside a block
        product("float32-odd", 77, 1000, 2832, "fp32"),
        # the largest: a long prompt's gate and up projections on the 32B shape
        product("prompt-4096-wide", 4096, 51200, 5120),
        # one token of each of 64 users of the 8B shape, whose last pages are partly filled
        cached("append-64", "append", 64, 1, 3000, 32, 8, 128, layout=1),
        # pieces of three prompts of the 8B shape, of unequal and odd lengths
        cached("append-prompts", "append", 3, 1500, 2000, 32, 8, 128, layout=2),
        # one user's answer on the 0.6B shape
        cached("decode-1", "decode", 1, 1, 700, 16, 8, 128, layout=3),
        # a server batch of the 8B shape, of unequal lengths
        cached("decode-48", "decode", 48, 1, 12000, 32, 8, 128, layout=4),
        # the 32-bit path with heads of 96 and no grouping
        cached("decode-float32", "decode", 5, 1, 1500, 16, 16, 96, "fp32", layout=5),
        # pieces of three prompts behind what they already hold
        cached("prompt-pieces", "prompt", 3, 900, 4000, 32, 8, 128, layout=6),
        # a long document's piece on the 8B shape
        cached("prompt-long", "prompt", 1, 4096, 8192, 32, 8, 128, layout=7),
    ]


def _spaced(rng, low: int, high: int) -> int:
    """A whole number between low and high, even over the logarithm."""
    return max(low, min(high, int(round(math.exp(rng.uniform(math.log(low), math.log(high + 0.49)))))))


def draw(rng) -> dict:
    most = {kind: max(sum(work(c).values()) for c in listed() if c["kind"] == kind) for kind in ("product", "append", "decode", "prompt")}
    while True:
        kind = rng.choice(("product", "product", "append", "decode", "decode", "prompt"))
        dtype = "fp32" if rng.random() < 0.2 else "bf16"
        if kind == "product":
            case = {"kind": kind, "rows": _spaced(rng, 1, 4096), "features": _spaced(rng, 100, 51200), "inputs": 16 * _spaced(rng, 12, 1600), "dtype": dtype}
        else:
            heads, kv_heads, dim = rng.choice(((16, 8, 128), (32, 8, 128), (64, 8, 128), (5, 5, 64), (6, 3, 48), (8, 1, 32), (16, 16, 96), (24, 4, 80), (40, 2, 64)))
            one = kind == "decode" or (kind == "append" and rng.random() < 0.5)
            case = {"kind": kind, "batch": _spaced(rng, 1, 128 if one else 6), "tokens": 1 if one else _spaced(rng, 1, 4096), "past": _spaced(rng, 1, 12000),
                    "heads": heads, "kv_heads": kv_heads, "head_dim": dim, "dtype": dtype, "layout": rng.randint(0, 1 << 20)}
            if dtype == "fp32" and case["tokens"] > 1 and kind == "prompt":
                case["tokens"], case["past"] = min(case["tokens"], 600), min(case["past"], 3000)
        if sum(work(case).values()) <= most[kind]:
            return case


# ----------------------------------------------------------------------------- sizes
def _lengths(case):
    """(this call's tokens, earlier tokens) of each sequence.  Of many sequences that answer, a few have ended: they have no keys at all."""
    rng = random.Random(case["layout"])
    tokens, past = [], []
    for i in range(case["batch"]):
        tokens.append(rng.randint(max(1, case["tokens"] // 3), case["tokens"]) if i else case["tokens"])
        past.append(rng.randint(case["past"] // 4, case["past"]) if i else case["past"])
        if case["kind"] == "decode" and i and rng.random() < 0.05:
            tokens[-1], past[-1] = 0, 0
    return tokens, past


def work(case) -> dict:
    size = 2 if case["dtype"] == "bf16" else 4
    if case["kind"] == "product":
        m, n, k = case["rows"], case["features"], case["inputs"]
        return {"bytes": (m * k + m * n) * size + n * k + 4 * -(-n // GROUP) * -(-k // GROUP), "flops": 2 * m * n * k}
    tokens, past = _lengths(case)
    heads, kv_heads, dim = case["heads"], case["kv_heads"], case["head_dim"]
    if case["kind"] == "append":
        # the projection in, queries, keys and values out; a rotation's angles
        return {"bytes": sum(tokens) * ((2 * heads + 2 * kv_heads) * dim * size + 2 * kv_heads * dim + 4 * dim), "flops": 10 * sum(tokens) * (heads + 2 * kv_heads) * dim}
    rows = case["batch"] if case["kind"] == "decode" else sum(tokens)
    seen = sum(n * p + n * (n + 1) // 2 for n, p in zip(tokens, past))
    held = sum(n + p for n, p in zip(tokens, past))
    return {"bytes": 2 * held * kv_heads * (dim + 4 / PAGE) + 2 * rows * heads * dim * size, "flops": 4 * heads * dim * seen}


# ----------------------------------------------------------------------------- inputs
def prepare(case, seed) -> dict:
    gen = torch.Generator(device="cuda")
    gen.manual_seed(seed)
    return _prepare_product(case, gen) if case["kind"] == "product" else _prepare_cached(case, gen, seed)


def _normal(gen, *shape):
    return torch.randn(shape, generator=gen, device="cuda")


def _prepare_product(case, gen) -> dict:
    """Rows as a norm leaves them, some columns far larger than the others; a weight whose blocks differ in size, as a checkpoint of such weights holds it."""
    m, n, k = case["rows"], case["features"], case["inputs"]
    dtype = TYPES[case["dtype"]]
    x = _normal(gen, m, k) * torch.where(torch.rand(k, generator=gen, device="cuda") < 0.01, 20.0, 1.0)
    blocks = (-(-n // GROUP), -(-k // GROUP))
    values = torch.empty((n, k), dtype=E4M3, device="cuda")
    values.copy_((_normal(gen, n, k) * 110.0).clamp_(-TOP, TOP))
    scales = 0.02 / 110.0 * torch.exp(0.5 * _normal(gen, *blocks))
    state = {"kind": "product", "x": x.to(dtype), "values": values, "scales": scales, "out": torch.empty((m, n), dtype=dtype, device="cuda")}
    if own:
        from qwen_triton_b200.ops import kernels
        state["weight"] = kernels.Fp8Weight(values, scales)
        state["scratch"] = kernels.fp8_rows(m, k, "cuda")
    return state


def _prepare_cached(case, gen, seed) -> dict:
    """A paged cache as the engine keeps it: pages in no order, their unused ends hold numbers; heads and pages differ in size."""
    tokens, past = _lengths(case)
    heads, kv_heads, dim, batch = case["heads"], case["kv_heads"], case["head_dim"], case["batch"]
    dtype = TYPES[case["dtype"]]
    counts = [-(-(n + p) // PAGE) for n, p in zip(tokens, past)]
    total = sum(counts) + 1
    order = list(range(total))
    random.Random(seed).shuffle(order)
    width = max(counts)
    table, at = [], 0
    for count in counts:
        table.append(order[at:at + count] + [order[-1]] * (width - count))
        at += count
    table = torch.tensor(table, dtype=torch.int32, device="cuda")
    held = {}
    for name in ("k", "v"):
        held[name] = torch.empty((total, kv_heads, PAGE, dim), dtype=E4M3, device="cuda")
        # a block's largest number lies between 224 and 448
        held[name].copy_((_normal(gen, total, kv_heads, PAGE, dim) * 85.0).clamp_(-TOP, TOP))
        held[name + "_scale"] = torch.exp2(torch.randint(-8, -5, (total, kv_heads), generator=gen, device="cuda").float())
    starts = [sum(tokens[:i]) for i in range(batch + 1)]
    state = {"kind": case["kind"], **held, "table": table, "heads": heads, "kv_heads": kv_heads, "dim": dim, "scale": dim ** -0.5, "dtype": dtype,
             "tokens_host": tokens, "past_host": past, "most": max(tokens), "seq_start": torch.tensor(starts, dtype=torch.int32, device="cuda"),
             "seq_past": torch.tensor(past, dtype=torch.int32, device="cuda"),
             "seq_len": torch.tensor([n + p for n, p in zip(tokens, past)], dtype=torch.int32, device="cuda")}
    if case["kind"] == "append":
        _prepare_append(state, gen, sum(tokens), tokens, past, starts)
    else:
        _prepare_queries(state, gen, batch if case["kind"] == "decode" else sum(tokens))
    if own:
        from qwen_triton_b200.ops import kernels
        state["cache"] = kernels.Cache8(state["k"], state["v"], state["k_scale"], state["v_scale"])
        if case["kind"] == "append":
            state["projection"] = kernels.GemmOut(state["qkv"][None])
        if case["kind"] == "decode":
            state["plan"] = kernels.decode8_plan(batch, num_heads=heads, num_kv_heads=kv_heads, head_dim=dim, dtype=dtype, max_context=max(n + p for n, p in zip(tokens, past)))
            state["part_acc"] = torch.empty(state["plan"].acc_elements, dtype=torch.float32, device="cuda")
            state["part_ml"] = torch.empty(state["plan"].ml_elements, dtype=torch.float32, device="cuda")
    return state


def _prepare_append(state, gen, rows, tokens, past, starts) -> None:
    heads, kv_heads, dim = state["heads"], state["kv_heads"], state["dim"]
    # projections have heads of different sizes; keys and queries pass a norm, values do not
    size = torch.exp(0.5 * _normal(gen, heads + 2 * kv_heads)).repeat_interleave(dim)
    state["qkv"] = (_normal(gen, rows, (heads + 2 * kv_heads) * dim) * size).to(state["dtype"])
    state["q_weight"], state["k_weight"] = 1.0 + 0.1 * _normal(gen, dim), 1.0 + 0.1 * _normal(gen, dim)
    longest = max(n + p for n, p in zip(tokens, past))
    inverse = 1e6 ** (-torch.arange(0, dim, 2, device="cuda").double() / dim)
    angle = torch.arange(longest, device="cuda").double()[:, None] * inverse
    state["cos_sin"] = torch.cat((angle.cos(), angle.sin()), 1).float()
    state["position"] = torch.tensor([p + j for n, p in zip(tokens, past) for j in range(n)], device="cuda")
    # the pages that are written: (sequence, page of the sequence, first place written, places written, first token)
    blocks = []
    for i, (n, p) in enumerate(zip(tokens, past)):
        for page in range(p // PAGE, -(-(p + n) // PAGE)):
            low, high = max(p, page * PAGE), min(p + n, (page + 1) * PAGE)
            blocks.append((i, page, low - page * PAGE, high - low, starts[i] + low - p))
    state["blocks"] = torch.tensor(blocks, device="cuda")
    state["q"] = torch.empty((rows, heads, dim), dtype=state["dtype"], device="cuda")


def _prepare_queries(state, gen, rows) -> None:
    """Queries that lean towards one key of what they see, as trained ones do."""
    heads, kv_heads, dim, device = state["heads"], state["kv_heads"], state["dim"], "cuda"
    q = _normal(gen, rows, heads, dim)
    pick = torch.rand((rows, heads), generator=gen, device=device)
    if state["kind"] == "decode":
        sequence, last = torch.arange(rows, device=device), state["seq_len"].long() - 1
    else:
        sequence = torch.repeat_interleave(torch.arange(len(state["tokens_host"]), device=device), torch.tensor(state["tokens_host"], device=device))
        last = state["seq_past"].long()[sequence] + torch.arange(rows, device=device) - state["seq_start"].long()[sequence]
    place = (pick * (last + 1)[:, None]).long().clamp(max=last.clamp(min=0)[:, None])
    page = torch.gather(state["table"].long()[sequence], 1, place // PAGE)
    kv_head = (torch.arange(heads, device=device) // (heads // kv_heads)).expand(rows, heads)
    key = state["k"].view(torch.uint8)[page, kv_head, place % PAGE].view(E4M3).float() * state["k_scale"][page, kv_head][..., None]
    state["q"] = (q + 0.5 * key).to(state["dtype"])
    state["out"] = torch.empty_like(state["q"])


# ----------------------------------------------------------------------------- one pass
def run(state):
    kind = state["kind"]
    if own:
        from qwen_triton_b200.ops import kernels
        if kind == "product":
            kernels.gemm_fp8(state["x"], state["weight"], state["out"], state["scratch"])
            return state["out"]
        if kind == "append":
            kernels.qkv_write_cache8(state["projection"], state["q"], state["cache"], state["seq_start"], state["seq_past"], state["table"], state["most"],
                                     state["q_weight"], state["k_weight"], EPS, state["cos_sin"])
            return {"q": state["q"], "k": state["k"], "v": state["v"], "k_scale": state["k_scale"], "v_scale": state["v_scale"]}
        if kind == "decode":
            kernels.attention_decode_cache8(state["q"], state["cache"], state["out"], state["table"], state["seq_len"], state["scale"], state["plan"],
                                            state["part_acc"], state["part_ml"])
        else:
            kernels.attention_prefill_cache8(state["q"], state["cache"], state["out"], state["table"], state["seq_start"], state["seq_past"], state["most"],
                                             state["scale"])
        return state["out"]
    return {"product": _plain_product, "append": _plain_append, "decode": _plain_decode, "prompt": _plain_prompt}[kind](state)


def _plain_product(state):
    x = state["x"].float()
    (m, k), n = x.shape, state["values"].shape[0]
    groups = -(-k // GROUP)
    pieces = torch.nn.functional.pad(x, (0, groups * GROUP - k)).view(m, groups, GROUP)
    x_scale = (pieces.abs().amax(2, keepdim=True) / TOP).clamp(min=2.0 ** -100)
    x8 = (pieces / x_scale).clamp(-TOP, TOP).to(E4M3)
    rows = (x8.float() * x_scale).view(m, -1)[:, :k]
    scale = state["scales"].repeat_interleave(GROUP, 0)[:n].repeat_interleave(GROUP, 1)[:, :k]
    return torch.matmul(rows, (state["values"].float() * scale).T).to(state["x"].dtype)


def _rotated(x, cos_sin, position):
    """x [tokens, heads, dim], pairs (i, i + dim / 2)."""
    cos, sin = cos_sin[position][:, None].chunk(2, dim=2)
    a, b = x.chunk(2, dim=2)
    return torch.cat((a * cos - b * sin, b * cos + a * sin), 2)


def _needed(largest):
    """The smallest e with largest <= 448 * 2^e, between -40 and 40."""
    part, power = torch.frexp(largest)
    return torch.where(largest == 0, -40, torch.where(part <= 0.875, power - 9, power - 8)).clamp(-40, 40)


def _plain_append(state):
    heads, kv_heads, dim = state["heads"], state["kv_heads"], state["dim"]
    q, k, v = state["qkv"].float().view(-1, heads + 2 * kv_heads, dim).split((heads, kv_heads, kv_heads), dim=1)
    q = q * torch.rsqrt(q.square().mean(2, keepdim=True) + EPS) * state["q_weight"]
    k = k * torch.rsqrt(k.square().mean(2, keepdim=True) + EPS) * state["k_weight"]
    q, k = _rotated(q, state["cos_sin"], state["position"]), _rotated(k, state["cos_sin"], state["position"])
    state["q"].copy_(q)
    sequence, page, first, count, token = state["blocks"].T
    page = state["table"].long()[sequence, page]
    place = torch.arange(PAGE, device=page.device)[None, :]
    new = (place >= first[:, None]) & (place < (first + count)[:, None])
    source = torch.where(new, token[:, None] + place - first[:, None], 0)
    new, kept = new[:, None, :, None], (place < first[:, None])[:, None, :, None]
    _plain_write(state, "k", k, page, source, new, kept, first)
    _plain_write(state, "v", v, page, source, new, kept, first)
    return {"q": state["q"], "k": state["k"], "v": state["v"], "k_scale": state["k_scale"], "v_scale": state["v_scale"]}


def _plain_write(state, name, rows, page, source, new, kept, first) -> None:
    rows = rows[source].permute(0, 2, 1, 3)                                            # [pages, kv_heads, 64, dim]
    largest = torch.where(new, rows.abs(), 0.0).amax((2, 3))
    was = torch.frexp(state[name + "_scale"][page])[1] - 1
    power = torch.where(first[:, None] == 0, _needed(largest), torch.maximum(was, _needed(largest)))
    held = state[name].view(torch.uint8)[page].view(E4M3)
    smaller = held.float() * torch.exp2((was - power).float())[:, :, None, None]
    written = (rows * torch.exp2(-power.float())[:, :, None, None]).clamp(-TOP, TOP)
    state[name].view(torch.uint8)[page] = torch.where(new, written, torch.where(kept, smaller, held.float())).to(E4M3).view(torch.uint8)
    state[name + "_scale"][page] = torch.exp2(power.float())


def _gathered(state, name):
    """[sequences, kv_heads, tokens, dim] in 32 bits, as long as the longest page list."""
    table = state["table"].long()
    held = state[name].view(torch.uint8)[table].view(E4M3).float() * state[name + "_scale"][table][..., None, None]
    return held.permute(0, 2, 1, 3, 4).flatten(2, 3)


def _plain_decode(state):
    batch, kv_heads, dim = len(state["tokens_host"]), state["kv_heads"], state["dim"]
    keys = _gathered(state, "k")
    q = state["q"].float().view(batch, kv_heads, -1, dim)
    scores = torch.matmul(q, keys.transpose(2, 3)) * state["scale"]
    visible = (torch.arange(keys.shape[2], device=q.device)[None, :] < state["seq_len"][:, None])[:, None, None]
    scores = scores.masked_fill(~visible, float("-inf"))
    top = scores.amax(3, keepdim=True)
    weights = torch.exp(scores - torch.where(top == float("-inf"), 0.0, top))
    total = weights.sum(3, keepdim=True)
    result = torch.matmul(weights, _gathered(state, "v"))
    return torch.where(total > 0, result / total, 0.0).view(batch, -1, dim).to(state["dtype"])


def _plain_prompt(state):
    batch, heads, kv_heads, dim, most = len(state["tokens_host"]), state["heads"], state["kv_heads"], state["dim"], state["most"]
    keys = _gathered(state, "k")
    place = torch.arange(most, device=keys.device)[None, :]
    count = (state["seq_start"][1:] - state["seq_start"][:-1])[:, None]
    row = torch.where(place < count, state["seq_start"][:-1, None] + place, 0).long()
    q = state["q"].float()[row].view(batch, most, kv_heads, -1, dim).permute(0, 2, 3, 1, 4)       # [sequences, kv_heads, group, queries, dim]
    group = heads // kv_heads
    scores = torch.matmul(q.reshape(batch, kv_heads, group * most, dim), keys.transpose(2, 3)).view(batch, kv_heads, group, most, -1)
    hidden = torch.arange(keys.shape[2], device=keys.device)[None, None, :] > (state["seq_past"][:, None] + place)[:, :, None]
    scores.mul_(state["scale"]).masked_fill_(hidden[:, None, None], float("-inf"))
    weights = scores.sub_(scores.amax(4, keepdim=True)).exp_()
    total = weights.sum(4, keepdim=True)
    result = torch.matmul(weights.view(batch, kv_heads, group * most, -1), _gathered(state, "v")).view(batch, kv_heads, group, most, dim) / total
    result = result.permute(0, 3, 1, 2, 4).reshape(batch, most, heads, dim)
    return result[(place < count)].to(state["dtype"])


# ----------------------------------------------------------------------------- in 64 bits
def exact(case, seed):
    state = prepare(case, seed)
    return {"product": _exact_product, "append": _exact_append, "decode": _exact_attention, "prompt": _exact_attention}[case["kind"]](state)


def _as_e4m3(x):
    """The nearest number of sign, 4 bits of exponent and 3 of mantissa, ties to the even one, in 64 bits."""
    exponent = (torch.frexp(x)[1] - 1).clamp(min=-6)
    step = torch.exp2(exponent.double() - 3)
    return ((x / step).round() * step).clamp(-TOP, TOP)


def _exact_product(state):
    x, k = state["x"], state["x"].shape[1]
    y = torch.zeros((x.shape[0], state["values"].shape[0]), dtype=torch.float64, device=x.device)
    by_row = torch.arange(y.shape[1], device=x.device) // GROUP
    for g in range(-(-k // GROUP)):
        columns = slice(g * GROUP, min(k, (g + 1) * GROUP))
        piece = x[:, columns].float()
        scale = torch.maximum(piece.abs().max(1).values / TOP, torch.full((), 2.0 ** -100, device=x.device))     # rounded to 32 bits, as it is kept
        rows = _as_e4m3((piece / scale[:, None]).double())                                                       # likewise
        y += scale.double()[:, None] * (rows @ state["values"][:, columns].double().T) * state["scales"][by_row, g].double()
    return y


def _scale_of(largest):
    """The smallest power of two whose 448-fold reaches `largest`, among 2^-40 to 2^40."""
    near = torch.log2(largest / TOP).round()                                           # off by one at most
    near = near - 1 + (TOP * torch.exp2(near - 1) < largest) + (TOP * torch.exp2(near) < largest).double()
    return torch.exp2(near.clamp(-40, 40))


def _exact_append(state):
    heads, kv_heads, dim = state["heads"], state["kv_heads"], state["dim"]
    x = state["qkv"].double().view(-1, heads + 2 * kv_heads, dim)
    half = dim // 2
    cos, sin = (t.double()[state["position"]][:, None] for t in (state["cos_sin"][:, :half], state["cos_sin"][:, half:]))

    def treated(y, weight):
        y = y / (y.square().mean(2, keepdim=True) + EPS).sqrt() * weight.double()
        return torch.cat((y[..., :half] * cos - y[..., half:] * sin, y[..., half:] * cos + y[..., :half] * sin), 2)

    answer = {"q": treated(x[:, :heads], state["q_weight"])}
    fresh = {"k": treated(x[:, heads:heads + kv_heads], state["k_weight"]), "v": x[:, heads + kv_heads:]}
    table = state["table"].tolist()
    for name in ("k", "v"):
        held, scale = state[name].double(), state[name + "_scale"].double()
        for i, page, first, count, token in state["blocks"].tolist():
            p = table[i][page]
            rows = fresh[name][token:token + count].transpose(0, 1)                                              # [kv_heads, count, dim]
            needed = _scale_of(rows.abs().amax((1, 2)))
            new = torch.maximum(needed, scale[p]) if first else needed
            if first:
                held[p, :, :first] *= (scale[p] / new)[:, None, None]
            held[p, :, first:first + count] = rows / new[:, None, None]
            scale[p] = new
        answer[name], answer[name + "_scale"] = held, scale
    return {name: answer[name] for name in ("q", "k", "v", "k_scale", "v_scale")}


def _exact_attention(state):
    """Each sequence by itself over its own page list."""
    q, kv_heads = state["q"].double(), state["kv_heads"]
    group, out, at = state["heads"] // kv_heads, torch.zeros_like(q), 0
    for i, (tokens, past) in enumerate(zip(state["tokens_host"], state["past_host"])):
        rows = slice(i, i + 1) if state["kind"] == "decode" else slice(at, at + tokens)
        at += tokens
        if not tokens:
            continue
        pages = state["table"][i, :-(-(tokens + past) // PAGE)].long()
        unseen = torch.arange(tokens + past, device=q.device)[None, :] > past + torch.arange(tokens, device=q.device)[:, None]
        for g in range(kv_heads):
            keys, values = ((state[name].view(torch.uint8)[pages, g].view(E4M3).double() * state[name + "_scale"][pages, g].double()[:, None, None]).flatten(0, 1)[:tokens + past]
                            for name in ("k", "v"))
            for h in range(g * group, (g + 1) * group):
                weights = torch.softmax((q[rows, h] @ keys.T * state["scale"]).masked_fill(unseen, -math.inf), dim=1)
                out[rows, h] = weights @ values
    return out
