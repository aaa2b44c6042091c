"""Two operators for several continuations of one prompt, as cases that can be timed and checked one by one.

* ``kind: "attention"``  one query token for each of ``batch`` sequences over a paged cache in which groups of sequences hold the same
  first pages: attention that reads a group's shared keys and values once for all of its members.
* ``kind: "sampling"``  one token per row of logits with a temperature, top-k, top-p and min-p of its own, from a given uniform
  number, and the log-probability with which it was drawn.

Lengths within a case follow from its ``layout`` number, so that a case says all of its sizes; the seed gives the numbers.
"""
from __future__ import annotations

import math
import random

import torch

own = False

PAGE = 64                     # tokens a page
UNITS = float(1 << 40)        # weights are added up as whole numbers in units of 2^-40 of the largest, so that no order of additions shows


# ----------------------------------------------------------------------------- cases
def listed() -> list[dict]:
    def attention(name, batch, groups, shared, own_tokens, heads, kv_heads, dim, dtype="bf16", layout=0):
        return {"name": name, "kind": "attention", "batch": batch, "groups": groups, "shared": shared, "own": own_tokens, "heads": heads,
                "kv_heads": kv_heads, "head_dim": dim, "dtype": dtype, "layout": layout}

    def sampling(name, rows, vocab, filters, allowed=1.0, ties=False):
        return {"name": name, "kind": "sampling", "rows": rows, "vocab": vocab, "filters": filters, "allowed": allowed, "ties": ties}

    return [
        # two drafts of one short answer on the 0.6B shape: the smallest call, where latency counts
        attention("drafts-2", 2, 1, 199, 40, 16, 8, 128, layout=1),
        # eight requests behind one system prompt on the 8B shape
        attention("system-prompt-8", 8, 1, 2048, 130, 32, 8, 128, layout=2),
        # a server batch of users with three system prompts of unequal, odd lengths, and some users with none
        attention("three-prompts-48", 48, 3, 5000, 700, 32, 8, 128, layout=3),
        # 64 continuations of a long document on the 8B shape
        attention("document-64", 64, 1, 16384, 512, 32, 8, 128, layout=4),
        # the largest: 128 continuations of a document near the model's longest context on the 32B shape
        attention("document-128-wide", 128, 1, 32000, 600, 64, 8, 128, layout=5),
        # heads of 64 without grouping, as one of the small configurations has them
        attention("heads-64", 20, 1, 1500, 90, 5, 5, 64, layout=6),
        # the 32-bit path: five continuations
        attention("float32-5", 5, 1, 900, 60, 16, 8, 128, "fp32", layout=7),
        # one user, the usual filters
        sampling("user-1", 1, 151936, "usual"),
        # a small batch, each row with parameters of its own, logits of few bits so that tokens tie
        sampling("mixed-8", 8, 151936, "mixed", ties=True),
        # 64 rows under a grammar that allows a part of the vocabulary
        sampling("grammar-64", 64, 151936, "mixed", allowed=0.02),
        # a full server batch
        sampling("server-256", 256, 151936, "mixed"),
        # many drafts of a small vocabulary of odd size
        sampling("small-vocabulary-100", 100, 503, "mixed"),
    ]


def _spaced(rng, low: int, high: int) -> int:
    """A whole number between low and high, even over the logarithm."""
    return max(low, min(high, int(round(math.exp(rng.uniform(math.log(low), math.log(high + 0.49)))))))


def draw(rng) -> dict:
    if rng.random() < 0.4:
        vocab = rng.choice((_spaced(rng, 200, 151936), 151936, 151936, rng.randint(100000, 151936)))
        return {"kind": "sampling", "rows": _spaced(rng, 1, 256), "vocab": vocab, "filters": rng.choice(("usual", "mixed", "mixed")),
                "allowed": rng.choice((1.0, 1.0, 0.3, 0.01)), "ties": rng.random() < 0.3}
    most = sum(work(listed()[4]).values())
    while True:
        dtype = "fp32" if rng.random() < 0.2 else "bf16"
        heads, kv_heads, dim = rng.choice(((16, 8, 128), (32, 8, 128), (64, 8, 128), (5, 5, 64), (6, 3, 48), (8, 1, 32), (16, 16, 96), (24, 4, 80)))
        batch = _spaced(rng, 1, 128 if dtype == "bf16" else 12)
        case = {"kind": "attention", "batch": batch, "groups": rng.randint(1, min(4, batch)), "shared": _spaced(rng, 1, 32000 if dtype == "bf16" else 2000),
                "own": _spaced(rng, 1, 1000 if dtype == "bf16" else 300), "heads": heads, "kv_heads": kv_heads, "head_dim": dim, "dtype": dtype,
                "layout": rng.randint(0, 1 << 20)}
        if sum(work(case).values()) <= most:
            return case


# ----------------------------------------------------------------------------- sizes
def _layout(case):
    """(members of each group, shared tokens of each group, own tokens of each sequence).  The first group's prefix is the longest; of several groups the
    last shares nothing.  Every sequence has at least the token that is being answered."""
    rng = random.Random(case["layout"])
    batch, groups = case["batch"], case["groups"]
    order = list(range(batch))
    if groups > 1:
        rng.shuffle(order)
    cuts = sorted(rng.sample(range(1, batch), groups - 1)) if groups > 1 else []
    members = [order[a:b] for a, b in zip([0] + cuts, cuts + [batch])]
    shared = [case["shared"]] + [0 if g == groups - 1 else rng.randint(1, case["shared"]) for g in range(1, groups)]
    own_tokens = [rng.randint(max(1, case["own"] // 4), case["own"]) for _ in range(batch)]
    return members, shared, own_tokens


def work(case) -> dict:
    if case["kind"] == "sampling":
        # a row read once, about one exponential and a handful of operations a token; parameters in, token and log-probability out
        return {"bytes": case["rows"] * (4 * case["vocab"] + 28), "flops": 8 * case["rows"] * case["vocab"]}
    members, shared, own_tokens = _layout(case)
    size = 2 if case["dtype"] == "bf16" else 4
    distinct = sum(shared) + sum(own_tokens)
    seen = sum(len(m) * s for m, s in zip(members, shared)) + sum(own_tokens)
    per_token = 2 * case["kv_heads"] * case["head_dim"] * size
    rows = case["batch"] * case["heads"] * case["head_dim"]
    return {"bytes": distinct * per_token + 2 * rows * size, "flops": 4 * case["heads"] * case["head_dim"] * seen}


# ----------------------------------------------------------------------------- inputs
def prepare(case, seed) -> dict:
    return _prepare_sampling(case, seed) if case["kind"] == "sampling" else _prepare_attention(case, seed)


def _prepare_attention(case, seed) -> dict:
    """A paged cache as the engine keeps it: a group's shared prefix fills pages that all of its members list first, the rest of the last shared page is
    each member's own where the prefix ends inside it (members then list a copy of that page).  Pages are in no order, and their unused ends hold numbers."""
    device = torch.device("cuda")
    dtype = torch.bfloat16 if case["dtype"] == "bf16" else torch.float32
    heads, kv_heads, dim, batch = case["heads"], case["kv_heads"], case["head_dim"], case["batch"]
    members, shared, own_tokens = _layout(case)
    lengths = [0] * batch
    tables = [[] for _ in range(batch)]
    total = 1 + sum(s // PAGE + sum(-(-(s + own_tokens[i]) // PAGE) - s // PAGE for i in m) for m, s in zip(members, shared))
    free = list(range(total))
    random.Random(seed).shuffle(free)
    copies = []                                              # (from, to): a partly shared page copied for a member
    share = []
    at = 0
    for group, tokens in zip(members, shared):
        whole = [free.pop() for _ in range(tokens // PAGE)]
        part = free.pop() if tokens % PAGE else None
        for number, i in enumerate(group):
            lengths[i] = tokens + own_tokens[i]
            pages = list(whole)
            if part is not None:
                page = part if number == 0 else free.pop()
                if number:
                    copies.append((part, page))
                pages.append(page)
            while len(pages) * PAGE < lengths[i]:
                pages.append(free.pop())
            tables[i] = pages
        share.append([at, len(group), tokens])
        at += len(group)
    width = max(len(t) for t in tables)
    table = torch.tensor([t + [0] * (width - len(t)) for t in tables], dtype=torch.int32, device=device)
    gen = torch.Generator(device=device)
    gen.manual_seed(seed)
    k_cache = torch.randn((total, kv_heads, PAGE, dim), generator=gen, device=device, dtype=dtype)
    v_cache = torch.randn((total, kv_heads, PAGE, dim), generator=gen, device=device, dtype=dtype)
    if copies:
        source = torch.tensor([a for a, _ in copies], device=device)
        target = torch.tensor([b for _, b in copies], device=device)
        k_cache[target] = k_cache[source]
        v_cache[target] = v_cache[source]
    # queries lean towards one key of what they see, as trained ones do
    q = torch.randn((batch, heads, dim), generator=gen, device=device)
    pick = torch.rand((batch, heads), generator=gen, device=device)
    length = torch.tensor(lengths, dtype=torch.int32, device=device)
    position = (pick * length[:, None]).long().clamp(max=(length.long() - 1)[:, None])
    page = torch.gather(table.long(), 1, position // PAGE)
    kv_head = torch.arange(heads, device=device) // (heads // kv_heads)
    q = (q + 0.5 * k_cache[page, kv_head[None, :], position % PAGE].float()).to(dtype)
    state = {"kind": "attention", "q": q, "k_cache": k_cache, "v_cache": v_cache, "table": table, "seq_len": length,
             "members": torch.tensor([i for m in members for i in m], dtype=torch.int32, device=device),
             "share": torch.tensor(share, dtype=torch.int32, device=device), "kv_heads": kv_heads, "scale": dim ** -0.5,
             "share_host": share, "members_host": members, "lengths_host": lengths, "out": torch.empty_like(q)}
    if own:
        from qwen_triton_b200.ops import kernels
        plan = kernels.shared_plan(batch, num_heads=heads, num_kv_heads=kv_heads, head_dim=dim, dtype=dtype, groups=len(members),
                                   most_members=max(len(m) for m in members), most_shared=max(shared), most_own=max(own_tokens))
        state["plan"] = plan
        state["part_acc"] = torch.empty(plan.acc_elements, dtype=torch.float32, device=device)
        state["part_ml"] = torch.empty(plan.ml_elements, dtype=torch.float32, device=device)
    return state


def _prepare_sampling(case, seed) -> dict:
    """Logits as a language model's head leaves them: a broad normal floor, a few hundred tokens that stand out, some rows sure of one token."""
    device = torch.device("cuda")
    rows, vocab = case["rows"], case["vocab"]
    gen = torch.Generator(device=device)
    gen.manual_seed(seed)
    rng = random.Random(seed)
    logits = 2.0 * torch.randn((rows, vocab), generator=gen, device=device)
    stands_out = torch.rand((rows, vocab), generator=gen, device=device) < max(300 / vocab, 1e-3) / 2
    logits += stands_out * (6.0 + 3.0 * torch.randn((rows, vocab), generator=gen, device=device))
    sure = torch.rand((rows, 1), generator=gen, device=device) < 0.3
    logits.scatter_add_(1, torch.randint(0, vocab, (rows, 1), generator=gen, device=device), 12.0 * sure.float())
    if case["ties"]:
        logits = logits.bfloat16().float()
    if case["allowed"] < 1.0:
        barred = torch.rand((rows, vocab), generator=gen, device=device) >= case["allowed"]
        logits.masked_fill_(barred, float("-inf"))
    temperature, top_k, top_p, min_p = [], [], [], []
    for row in range(rows):
        if case["filters"] == "usual":
            temperature.append(0.7), top_k.append(50), top_p.append(0.9), min_p.append(0.02)
            continue
        temperature.append(rng.choice((0.0, 0.6, 0.7, 0.8, 1.0, 1.0)))
        top_k.append(rng.choice((0, 0, 1, 20, 50, 400)))
        top_p.append(rng.choice((1.0, 0.95, 0.9, 0.8)))
        min_p.append(rng.choice((0.0, 0.0, 0.02, 0.1)))
    def vector(values, dtype):
        return torch.tensor(values, dtype=dtype, device=device)
    return {"kind": "sampling", "logits": logits, "temperature": vector(temperature, torch.float32), "top_k": vector(top_k, torch.int32),
            "top_p": vector(top_p, torch.float32), "min_p": vector(min_p, torch.float32),
            "uniform": torch.rand(rows, generator=gen, device=device), "tokens": torch.empty(rows, dtype=torch.int32, device=device),
            "logprob": torch.empty(rows, dtype=torch.float32, device=device)}


# ----------------------------------------------------------------------------- one pass
def run(state):
    if own:
        from qwen_triton_b200.ops import kernels
        if state["kind"] == "attention":
            kernels.attention_decode_shared(state["q"], state["k_cache"], state["v_cache"], state["out"], state["table"], state["seq_len"],
                                            state["members"], state["share"], state["kv_heads"], PAGE, state["scale"], state["plan"],
                                            state["part_acc"], state["part_ml"])
            return state["out"]
        kernels.sample_filtered(state["logits"], state["temperature"], state["top_k"], state["top_p"], state["min_p"], state["uniform"],
                                state["tokens"], state["logprob"])
        return {"tokens": state["tokens"], "logprob": state["logprob"]}
    return _plain_sampling(state) if state["kind"] == "sampling" else _plain_attention(state)


def _rows_of(cache, pages, tokens):
    """[tokens, kv_heads, dim] in float from a page list."""
    return cache[pages[:-(-tokens // PAGE)].long()].permute(0, 2, 1, 3).reshape(-1, cache.shape[1], cache.shape[3])[:tokens].float()


def _plain_attention(state):
    q, k_cache, v_cache, table = state["q"], state["k_cache"], state["v_cache"], state["table"]
    kv_heads, scale = state["kv_heads"], state["scale"]
    batch, heads, dim = q.shape
    per = heads // kv_heads
    out = torch.empty_like(q)
    for group, (_, _, shared) in zip(state["members_host"], state["share_host"]):
        rows = torch.tensor(group, device=q.device)
        n = len(group)
        queries = q[rows].float().reshape(n, kv_heads, per, dim)
        by_head = queries.permute(1, 0, 2, 3).reshape(kv_heads, n * per, dim)
        most_own = max(state["lengths_host"][i] for i in group) - shared
        # the shared keys once for all members
        keys = _rows_of(k_cache, table[group[0]], shared)
        scores = torch.matmul(by_head, keys.permute(1, 2, 0)).reshape(kv_heads, n, per, shared) * scale
        # every member's own keys, padded to the longest
        place = shared + torch.arange(most_own, device=q.device)
        visible = place[None, :] < state["seq_len"][rows][:, None]
        place = torch.where(visible, place[None, :], 0)
        page = torch.gather(table[rows].long(), 1, place // PAGE)
        own_keys = k_cache[page, :, place % PAGE].float()                                  # [n, own, kv_heads, dim]
        own_scores = torch.matmul(queries.permute(1, 0, 2, 3), own_keys.permute(2, 0, 3, 1)) * scale
        own_scores = own_scores.masked_fill(~visible[None, :, None, :], float("-inf"))
        top = own_scores.amax(-1, keepdim=True)
        if shared:
            top = torch.maximum(top, scores.amax(-1, keepdim=True))
        own_weights = torch.exp(own_scores - top)
        total = own_weights.sum(-1, keepdim=True)
        own_values = v_cache[page, :, place % PAGE].float().masked_fill(~visible[:, :, None, None], 0.0)
        result = torch.matmul(own_weights, own_values.permute(2, 0, 1, 3))                 # [kv_heads, n, per, dim]
        if shared:
            weights = torch.exp(scores - top)
            total = total + weights.sum(-1, keepdim=True)
            values = _rows_of(v_cache, table[group[0]], shared)
            result = result + torch.matmul(weights.reshape(kv_heads, n * per, shared), values.permute(1, 0, 2)).reshape(kv_heads, n, per, dim)
        out[rows] = (result / total).permute(1, 0, 2, 3).reshape(n, heads, dim).to(q.dtype)
    return out


def _plain_sampling(state):
    logits = state["logits"]
    rows, vocab = logits.shape
    temperature, uniform = state["temperature"][:, None], state["uniform"][:, None]
    top = logits.amax(1, keepdim=True)
    greedy = temperature <= 0
    depth = torch.where(logits == top, 0.0, logits - top) / torch.where(greedy, 1.0, temperature)
    weight = torch.exp(depth)
    units = (weight * UNITS).round().long()
    # how many tokens, and what mass of the kept ones, lie strictly above each token: over the sorted row, at the first of its equals
    ordered, order = torch.sort(logits, dim=1, descending=True)
    first = torch.searchsorted(-ordered, -ordered)
    above = torch.empty_like(first).scatter_(1, order, first)
    top_k = state["top_k"][:, None].long()
    kept = (above < top_k) | (top_k <= 0)
    sorted_units = torch.gather(torch.where(kept, units, 0), 1, order)
    before = torch.gather(torch.cumsum(sorted_units, 1) - sorted_units, 1, first)
    mass_above = torch.empty_like(before).scatter_(1, order, before)
    mass = sorted_units.sum(1, keepdim=True)
    top_p = state["top_p"][:, None]
    kept &= (mass_above.double() < top_p.double() * mass.double()) | (top_p >= 1)
    kept &= weight >= state["min_p"][:, None].clamp(max=1.0)
    running = torch.cumsum(torch.where(kept, units, 0), 1)
    total = running[:, -1:]
    target = (uniform.double() * total.double()).floor().long()
    token = (running > target).to(torch.uint8).argmax(1, keepdim=True)
    logprob = torch.gather(depth, 1, token) - torch.log(total.float() / UNITS)
    token = torch.where(greedy, (logits == top).to(torch.uint8).argmax(1, keepdim=True), token)
    logprob = torch.where(greedy, 0.0, logprob)
    nothing = top == float("-inf")
    return {"tokens": torch.where(nothing, 0, token)[:, 0].int(), "logprob": torch.where(nothing, float("-inf"), logprob)[:, 0]}


# ----------------------------------------------------------------------------- in 64 bits
def exact(case, seed):
    state = prepare(case, seed)
    return _exact_sampling(state) if case["kind"] == "sampling" else _exact_attention(state)


def _exact_attention(state):
    """Each sequence by itself over its own page list, without a word of what is shared."""
    q = state["q"].double()
    batch, heads, dim = q.shape
    per = heads // state["kv_heads"]
    out = torch.empty_like(q)
    for i, length in enumerate(state["lengths_host"]):
        places = torch.arange(length, device=q.device)
        page, slot = state["table"][i].long()[places // PAGE], places % PAGE
        for g in range(state["kv_heads"]):
            keys, values = state["k_cache"][page, g, slot].double(), state["v_cache"][page, g, slot].double()
            weights = torch.softmax(state["scale"] * (q[i, g * per:(g + 1) * per] @ keys.T), dim=1)
            out[i, g * per:(g + 1) * per] = weights @ values
    return out


def _exact_sampling(state):
    tokens, logprobs = [], []
    for row in range(state["logits"].shape[0]):
        x = state["logits"][row].double()
        temperature, k = float(state["temperature"][row]), int(state["top_k"][row])
        p, m, u = float(state["top_p"][row]), float(state["min_p"][row]), float(state["uniform"][row])
        best = float(x.max())
        if best == -math.inf:
            tokens.append(0), logprobs.append(-math.inf)
            continue
        if temperature <= 0:
            tokens.append(int((x == best).nonzero()[0])), logprobs.append(0.0)
            continue
        y = (x - best) / temperature
        w = y.exp()
        floor = -math.inf
        if 0 < k < x.numel():
            floor = float(x.topk(k).values[-1])
        if p < 1:
            values, counts = x[x >= floor].unique(return_counts=True)      # the distinct logits that are kept, ascending
            mass = ((values - best) / temperature).exp() * counts
            over = mass.flip(0).cumsum(0).flip(0) - mass                   # of strictly larger ones
            floor = float(values[over < p * mass.sum()].min())
        kept = (x >= floor) & (w >= m)
        running = torch.where(kept, w, 0.0).cumsum(0)
        token = int((running > u * running[-1]).nonzero()[0])
        tokens.append(token), logprobs.append(float(y[token] - running[-1].log()))
    device = state["logits"].device
    return {"tokens": torch.tensor(tokens, dtype=torch.int32, device=device), "logprob": torch.tensor(logprobs, dtype=torch.float64, device=device)}
