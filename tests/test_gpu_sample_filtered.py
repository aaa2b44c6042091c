"""Sampling under filters, a row's own parameters and given numbers, against a plain statement in 64 bits."""
from __future__ import annotations

import math

import pytest
import torch

from qwen_triton_b200.ops import kernels
from qwen_triton_b200.ops.kernels import KernelError

pytestmark = pytest.mark.gpu


def kept_of(x, temperature, k, p, m):
    """(weights that stay, else 0; y) of one row in 64 bits on the host, from the definition token by token over the distinct logits."""
    x = torch.where(x.isnan(), float("-inf"), x).double()
    best = x.max()
    y = torch.where(x == best, 0.0, x - best) / temperature
    w = y.exp()
    values, inverse, counts = x.unique(return_inverse=True, return_counts=True)
    above = (counts.flip(0).cumsum(0).flip(0) - counts)[inverse]
    kept = (above < k) if k > 0 else torch.ones_like(x, dtype=torch.bool)
    mass = torch.zeros_like(values).scatter_add_(0, inverse, torch.where(kept, w, 0.0))
    above_mass = (mass.flip(0).cumsum(0).flip(0) - mass)[inverse]
    if p < 1:
        kept &= above_mass < p * mass.sum()
    kept &= w >= min(m, 1.0)
    return torch.where(kept, w, 0.0), y


def settled(x, temperature, k, p, m):
    """(p, m) moved to where no rounding decides: p into the middle of the two running masses around it, m between two weights."""
    w, _ = kept_of(x, temperature, k, 1.0, 0.0)
    if p < 1:
        values, inverse = x.double().unique(return_inverse=True)
        mass = torch.zeros_like(values).scatter_add_(0, inverse, w).flip(0).cumsum(0) / w.sum()
        i = int((mass < p).sum())
        p = (float(mass[i - 1] if i else 0.0) + float(mass[min(i, len(mass) - 1)])) / 2
    if 0 < m < 1:
        ordered = w[w > 0].unique()
        i = int((ordered < m).sum())
        m = (float(ordered[i - 1] if i else 0.0) + float(ordered[min(i, len(ordered) - 1)])) / 2
    return p, m


def middle(weights, gen):
    """(token, number): a token that stays, by its weight, and a number in the middle of its part of the line, where that part is wide enough for a
    float and the sums' roundings to keep the number inside it."""
    running = weights.cumsum(0)
    total = float(running[-1])
    for _ in range(200):
        u = float(torch.rand((), generator=gen, dtype=torch.float64))
        token = int((running > u * total).nonzero()[0])
        low, high = float(running[token] - weights[token]) / total, float(running[token]) / total
        if high - low > 2.0 ** -16:
            return token, (low + high) / 2
    token = int(weights.argmax())
    return token, (float(running[token]) - 0.5 * float(weights[token])) / total


def run(logits, temperature, top_k, top_p, min_p, uniform, want_logprob=True):
    rows = logits.shape[0]
    def vector(values, dtype):
        return torch.tensor(values, dtype=dtype, device="cuda")
    out = torch.full((rows,), -5, dtype=torch.int32, device="cuda")
    logprob = torch.full((rows,), 9.0, device="cuda") if want_logprob else None
    kernels.sample_filtered(logits, vector(temperature, torch.float32), vector(top_k, torch.int32), vector(top_p, torch.float32),
                            vector(min_p, torch.float32), vector(uniform, torch.float32), out, logprob)
    return out.cpu(), None if logprob is None else logprob.cpu()


def check(logits, params, seed):
    """Rows with params[(T, k, p, m)] each: the token of the middle of its part, and its log-probability.  The logarithm's error: y is one subtraction and
    one division (2^-23 of |y|), the mass a sum whose terms have relative errors of a few 2^-24 times (1 + |y|), the logarithm 2^-22 of itself."""
    gen = torch.Generator().manual_seed(seed)
    rows = []
    for x, (t, k, p, m) in zip(logits.cpu(), params):
        p, m = settled(x, t, k, p, m)
        weights, y = kept_of(x, t, k, p, m)
        token, u = middle(weights, gen)
        rows.append((t, k, p, m, u, token, float(y[token] - weights.sum().log()), float(y[token])))
    tokens, logprob = run(logits, *[[r[c] for r in rows] for c in range(5)])
    assert tokens.tolist() == [r[5] for r in rows]
    for got, (_, _, _, _, _, _, want, y) in zip(logprob.tolist(), rows):
        assert abs(got - want) <= 2e-6 * (1 + abs(y) + abs(want)), (got, want)


PARAMS = [(1.0, 0, 1.0, 0.0), (0.7, 50, 1.0, 0.0), (0.8, 0, 0.9, 0.0), (1.0, 0, 1.0, 0.05), (1.3, 20, 0.95, 0.02), (0.3, 1, 0.5, 0.5), (2.5, 0, 0.999, 0.0),
          (1.0, 3, 0.7, 0.0), (0.05, 0, 0.9, 0.1), (5.0, 400, 0.99, 0.001), (1.0, 100000, 0.8, 0.0), (1.0, 7, 1.0, 0.9)]


@pytest.mark.parametrize("vocab", [1, 2, 31, 33, 199, 503, 1024, 4099, 32000, 50257, 151936, 151937, 262144, 500001])
def test_every_filter_at_many_sizes(vocab):
    gen = torch.Generator().manual_seed(vocab)
    logits = 2.5 * torch.randn((len(PARAMS), vocab), generator=gen)
    logits[:, torch.randint(0, vocab, (min(vocab, 40),), generator=gen)] += 6.0
    check(logits.cuda(), [(t, min(k, vocab), p, m) for t, k, p, m in PARAMS], vocab)


@pytest.mark.parametrize("step", [1.0, 0.25, 2.0 ** -4])
def test_tokens_that_tie_share_their_fate(step):
    gen = torch.Generator().manual_seed(int(step * 16))
    logits = (torch.randn((len(PARAMS), 5000), generator=gen) * 3 / step).round() * step
    logits[0, 100:200] = -0.0
    logits[0, 200:300] = 0.0
    check(logits.cuda(), PARAMS, 1)


def test_all_alike_and_nearly_alike():
    gen = torch.Generator().manual_seed(2)
    rows = torch.cat([torch.full((3, 40000), 1.5), 3.0 + 1e-4 * torch.rand((4, 40000), generator=gen), torch.full((1, 40000), -3.0e38)])
    check(rows.cuda(), [(1.0, 0, 1.0, 0.0), (1.0, 5, 0.5, 0.0), (0.5, 0, 0.5, 0.3), (1.0, 0, 0.5, 0.0), (1.0, 1000, 1.0, 0.0), (1.0, 20000, 0.25, 0.0),
                        (0.01, 0, 0.9, 0.999), (1.0, 0, 1.0, 0.0)], 3)


def test_barred_tokens():
    """Masks of -inf, of the lowest float and of NaN, down to one token that is left."""
    gen = torch.Generator().manual_seed(4)
    logits = 2 * torch.randn((len(PARAMS), 20001), generator=gen)
    for row, mask in enumerate((float("-inf"), torch.finfo(torch.float32).min, float("nan")) * 4):
        allowed = (1, 2, 30, 3000)[row // 3]
        barred = torch.randperm(20001, generator=gen)[allowed:]
        logits[row, barred] = mask
    check(logits.cuda(), PARAMS, 5)


def test_infinities_and_rows_that_leave_nothing():
    logits = torch.zeros((6, 1000))
    logits[0] = float("-inf")
    logits[1] = float("nan")
    logits[2, 500:] = float("inf")
    logits[3, 70] = float("inf")
    logits[4] = float("-inf")
    logits[5, 3] = float("nan")
    tokens, logprob = run(logits.cuda(), [1.0, 0.7, 1.0, 0.5, 0.0, 0.0], [0, 5, 0, 0, 0, 0], [1.0, 0.9, 0.9, 1.0, 1.0, 1.0], [0.0] * 6,
                          [0.5, 0.2, 0.0, 0.99, 0.1, 0.1])
    assert tokens.tolist() == [0, 0, 500, 70, 0, 0]
    assert logprob[:2].tolist() == [-math.inf] * 2 and logprob[4] == -math.inf
    assert abs(float(logprob[2]) + math.log(500)) < 1e-5 and logprob[3] == 0 and logprob[5] == 0


def test_greedy_rows_take_the_lowest_id():
    gen = torch.Generator().manual_seed(6)
    logits = torch.randn((5, 9999), generator=gen).round()
    tokens, logprob = run(logits.cuda(), [0.0, 0.0, -1.0, float("nan"), 0.0], [0, 3, 0, 0, 1], [1.0, 0.5, 1.0, 1.0, 0.1], [0.0, 0.1, 0.0, 0.0, 0.9], [0.3] * 5)
    assert tokens.tolist() == [int((row == row.max()).nonzero()[0]) for row in logits]
    assert logprob.tolist() == [0.0] * 5


def test_numbers_at_the_ends_and_parameters_beyond_theirs():
    """u = 0 gives the first token that stays, u at and beyond 1 the last; top_p <= 0 leaves the likeliest, min_p > 1 too."""
    logits = torch.tensor([[1.0, 5.0, 4.9, -3.0, 4.8, 5.0, -40.0]]).repeat(8, 1).cuda()
    tokens, _ = run(logits, [1.0] * 8, [3, 3, 3, 0, 0, 99, -4, 0], [1.0, 1.0, 1.0, 0.0, -1.0, 1.0, 2.0, 1.0], [0.0, 0.0, 0.0, 0.0, 0.0, 0.0, 0.0, 7.0],
                    [0.0, 1.0, 3.0, 0.999, 0.0, 0.0, 0.0, 0.999])
    assert tokens.tolist() == [1, 5, 5, 5, 1, 0, 0, 5]


def test_rows_apart_and_odd_addresses():
    """A part of wider rows, from an address that no wide load takes."""
    gen = torch.Generator().manual_seed(7)
    wide = 2 * torch.randn((len(PARAMS), 12345), generator=gen).cuda()
    view = wide[:, 3:10000]
    check(view, PARAMS, 8)
    check(wide[::2, 1:1002], PARAMS[::2], 9)


@pytest.mark.parametrize("vocab", [6000, 151936])
def test_heads_that_fit_no_list(vocab):
    """Flat rows: what stays is a large part of the vocabulary, by count, by mass and by both."""
    gen = torch.Generator().manual_seed(vocab)
    params = [(1.0, vocab // 2, 1.0, 0.0), (1.0, 0, 0.9, 0.0), (1.0, vocab // 3, 0.9, 0.0), (3.0, 0, 0.99, 0.02), (0.9, vocab - 1, 0.5, 0.0), (1.0, 5000, 0.99, 0.0),
              (2.0, 2500, 1.0, 0.0), (1e-3, 3000, 0.999, 0.0), (1e4, 0, 0.3, 0.0), (1.0, 0, 1.0, 1e-4), (1.0, 3000, 1.0, 1e-9), (50.0, 0, 0.5, 0.9)]
    logits = torch.randn((len(params), vocab), generator=gen)
    logits[::2] = (logits[::2] * 8).round() / 8               # hundreds of tokens to a value
    check(logits.cuda(), params, vocab)


def test_tokens_that_stand_out_side_by_side():
    """More of them in one block's part of the row than a part of the list holds, and all of them in one thread's."""
    logits = torch.randn((4, 151936), generator=torch.Generator().manual_seed(12)) - 20
    logits[0, 1000:1700] += 25
    logits[1, 40000:40004] += 25
    logits[2, 151900:] += 30
    logits[3, :300] += 25
    check(logits.cuda(), [(1.0, 500, 1.0, 0.0), (1.0, 3, 1.0, 0.0), (1.0, 0, 0.9, 0.0), (0.8, 299, 0.95, 0.001)], 13)


@pytest.mark.parametrize("rows, vocab", [(90, 40001), (330, 20003), (75, 151936), (40, 70000), (700, 8300)])
def test_more_rows_than_fit_at_a_time(rows, vocab):
    """Few blocks a row, rows that are left to a second launch: without filters, with wide heads, and none of these side by side with rows of every kind."""
    gen = torch.Generator().manual_seed(rows)
    logits = 2.0 * torch.randn((rows, vocab + 3), generator=gen)[:, 3:]
    logits[:, torch.randint(0, vocab, (30,), generator=gen)] += 7.0
    logits[1::5, ::3] = float("-inf")
    logits[2::5, 1::4] = float("nan")
    kinds = PARAMS + [(1.0, 0, 0.97, 0.0), (1.5, 0, 0.6, 1e-4), (2.0, 3000, 1.0, 0.0), (1.0, 900, 0.95, 0.0), (1e-6, 0, 1.0, 0.0)]
    params = [kinds[i % len(kinds)] for i in range(rows)]
    whole = torch.empty((rows, vocab + 3), device="cuda")
    whole[:, 3:] = logits.cuda()
    check(whole[:, 3:], params, rows + 1)
    nothing = torch.full((rows, vocab), float("-inf"), device="cuda")
    tokens, logprob = run(nothing, *[[p[c] for p in params] for c in range(4)], [0.5] * rows)
    assert tokens.tolist() == [0] * rows and logprob.tolist() == [-math.inf] * rows


@pytest.mark.parametrize("rows", [12, 156])
def test_shares_that_end_beside_a_token(rows):
    """top_p a millionth more or less than what lies before a token.  The weights' errors are 2^-23 and less of each, of both signs; what stays beside ten tokens that stand out is
    2e-5 of the mass: a millionth decides."""
    gen = torch.Generator().manual_seed(rows)
    vocab = 30000
    logits = torch.randn((rows, vocab), generator=gen).clamp(max=2.0)
    params, wanted = [], []
    for row in range(rows):
        heads = torch.randperm(vocab, generator=gen)[:10]
        logits[row, heads] = 22.0 + torch.rand((10,), generator=gen)
        w, _ = kept_of(logits[row], 1.0, 0, 1.0, 0.0)
        share = w[w > 0.1].sort(descending=True).values.cumsum(0) / w.sum()
        p = torch.tensor(float(share[1 + row % 8]) + (1e-6 if row % 2 else -1e-6)).item()
        weights, y = kept_of(logits[row], 1.0, 0, p, 0.0)
        token, u = middle(weights, gen)
        params.append((1.0, 0, p, 0.0, u))
        wanted.append((token, float(y[token] - weights.sum().log())))
    tokens, logprob = run(logits.cuda(), *[[p[c] for p in params] for c in range(5)])
    assert tokens.tolist() == [w[0] for w in wanted]
    for got, (_, want) in zip(logprob.tolist(), wanted):
        assert abs(got - want) <= 2e-6 * (3 + abs(want)), (got, want)


def test_no_order_of_additions_shows_and_the_stream_is_followed():
    gen = torch.Generator(device="cuda").manual_seed(8)
    logits = torch.randn((64, 151936), generator=gen, device="cuda")
    args = ([0.9] * 64, [0, 50] * 32, [0.95, 1.0, 0.7, 1.0] * 16, [0.0] * 64, [i / 64 for i in range(64)])
    tokens, logprob = run(logits, *args)
    again, logprob2 = run(logits, *args)
    assert torch.equal(tokens, again) and torch.equal(logprob, logprob2)
    stream = torch.cuda.Stream()
    late = torch.zeros_like(logits)
    torch.cuda.synchronize()
    with torch.cuda.stream(stream):
        torch.cuda._sleep(2_000_000)
        late.copy_(logits)
        third, _ = run(late, *args, want_logprob=False)
    assert torch.equal(tokens, third)


def test_shares_of_many_numbers():
    """Over an even grid of numbers each token comes as often as its weight says, to one grid step."""
    logits = torch.tensor([0.0, 1.0, 2.0, -1.0, 2.0, 0.5]).log_softmax(0)
    n = 4096
    tokens, _ = run(logits.repeat(n, 1).cuda(), [1.0] * n, [0] * n, [1.0] * n, [0.0] * n, [(i + 0.5) / n for i in range(n)])
    counts = torch.bincount(tokens, minlength=6).double()
    assert bool(((counts - n * logits.double().exp()).abs() <= 1).all())


def test_no_rows_and_refusals():
    empty = torch.empty((0, 50), device="cuda")
    run(empty, [], [], [], [], [])
    logits = torch.zeros((3, 50), device="cuda")
    f, k, out = torch.ones(3, device="cuda"), torch.zeros(3, dtype=torch.int32, device="cuda"), torch.zeros(3, dtype=torch.int32, device="cuda")
    good = dict(logits=logits, temperature=f, top_k=k, top_p=f, min_p=f, uniform=f, out=out, logprob=None)
    for changes, words in ((dict(logits=logits.cpu()), "CUDA"), (dict(logits=logits.bfloat16()), "float32"), (dict(logits=logits[0]), "rows"),
                           (dict(logits=logits.t()), "strides|shape"), (dict(logits=logits[:1].expand(3, 50)), "strides"),
                           (dict(logits=torch.zeros((3, 0), device="cuda")), "logits"), (dict(temperature=f[:2]), "temperature"),
                           (dict(top_k=f), "top_k"), (dict(top_p=f.double()), "top_p"), (dict(min_p=f.cpu()), "min_p"), (dict(uniform=f[::2]), "uniform"),
                           (dict(out=f), "out"), (dict(logprob=out), "logprob")):
        with pytest.raises(KernelError, match=words):
            kernels.sample_filtered(**{**good, **changes})


def test_the_largest_vocabulary_and_one_beyond():
    """2^23 equal logits weigh 2^63 units of 2^-40; a row of 2^24 would not fit 64 bits, so no more than the first are taken."""
    vocab = 1 << 23
    logits = torch.zeros((1, vocab + 1), device="cuda")
    for filters in ((0, 1.0, 0.0), (5, 0.5, 0.3)):            # ties share their fate: every token stays
        for u in (0.0, 0.25, 0.8125, 1.0):
            tokens, logprob = run(logits[:, :vocab], [1.0], [filters[0]], [filters[1]], [filters[2]], [u])
            assert tokens.tolist() == [min(int(u * vocab), vocab - 1)]
            assert abs(float(logprob[0]) + math.log(vocab)) <= 2e-6 * (1 + math.log(vocab))
    with pytest.raises(KernelError, match="vocabulary"):
        run(logits, [1.0], [0], [1.0], [0.0], [0.5])


def test_a_share_that_the_tail_of_a_large_vocabulary_decides():
    """Masses are sums of whole units of 2^-40.  2^23 - 2 tokens of 1.55 units count as two each, 3.4e-6 of the mass more than their weights: with those, what lies
    before the second token is p of the mass and 6e-7 more, with the weights 2.5e-6 less.  However the row is walked (top_k, which leaves every token
    here, takes another way), the units decide."""
    vocab = 1 << 23
    logits = torch.full((1, vocab), math.log(1.55) - 40 * math.log(2))
    first, second = 1000, vocab - 77
    logits[0, first], logits[0, second] = 0.0, math.log(0.1)
    p = 1 / ((1.1 + (vocab - 2) * 1.55 * 2.0 ** -40) * (1 + 2.5e-6))
    assert p * (1.1 + (vocab - 2) * 2 * 2.0 ** -40) > 1 + 5e-7
    for k in (0, vocab - 1):
        tokens, logprob = run(logits.cuda(), [1.0], [k], [p], [0.0], [0.97])
        assert tokens.tolist() == [second]
        assert abs(float(logprob[0]) - math.log(0.1 / 1.1)) < 1e-5


def test_shares_that_end_beside_a_token_of_a_large_vocabulary():
    """As above, over two million tokens whose units' roundings cancel: a millionth more or less decides."""
    gen = torch.Generator().manual_seed(21)
    vocab = 1 << 21
    for row in range(4):
        logits = torch.randn((1, vocab), generator=gen).clamp(max=2.0)
        heads = torch.randperm(vocab, generator=gen)[:10]
        logits[0, heads] = 26.0 + torch.rand((10,), generator=gen)
        w, _ = kept_of(logits[0], 1.0, 0, 1.0, 0.0)
        share = w[w > 0.1].sort(descending=True).values.cumsum(0) / w.sum()
        p = torch.tensor(float(share[1 + 2 * row]) + (1e-6 if row % 2 else -1e-6)).item()
        weights, y = kept_of(logits[0], 1.0, 0, p, 0.0)
        token, u = middle(weights, gen)
        tokens, logprob = run(logits.cuda(), [1.0], [0], [p], [0.0], [u])
        want = float(y[token] - weights.sum().log())
        assert tokens.tolist() == [token]
        assert abs(float(logprob[0]) - want) <= 2e-6 * (3 + abs(want))


@pytest.mark.parametrize("vocab", [600, 5000, 40000])
def test_weights_that_round_to_the_least_stay_whichever_way_the_row_goes(vocab):
    """At a temperature of 10,000 a logit 1e-4 below the largest weighs 1 - 1e-8, which is 1 in 32 bits: min_p = 1 keeps both, and a top_k that leaves every token
    (which makes the row go another way) changes nothing."""
    logits = torch.full((1, vocab), -30.0)
    logits[0, 7], logits[0, vocab // 2] = 0.03, 0.03 - 1e-4
    for u, token in ((0.2, 7), (0.8, vocab // 2)):
        for k in (0, vocab - 1):
            tokens, logprob = run(logits.cuda(), [1e4], [k], [1.0], [1.0], [u])
            assert tokens.tolist() == [token] and abs(float(logprob[0]) + math.log(2)) < 1e-6
