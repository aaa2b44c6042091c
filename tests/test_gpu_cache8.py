"""A cache of keys and values in 8 bits: the write from a projection, attention of single tokens and of prompts over it, against 64 bits."""
import math

import pytest
import torch

import plain_8bit as plain

pytestmark = pytest.mark.gpu
E4M3 = torch.float8_e4m3fn
PAGE = 64
BF16, F32 = torch.bfloat16, torch.float32
# heads, kv heads, head size: grouped, not grouped, one kv head, many rows a kv head, sizes that no power of two has
HEADS = [(32, 8, 128), (16, 16, 96), (5, 5, 64), (6, 3, 48), (8, 1, 32), (24, 4, 80), (40, 2, 64), (4, 2, 16), (4, 2, 256), (3, 1, 160)]


def _filled(pages, kv_heads, dim, seed, spread=3):
    """A cache with numbers everywhere, under scales that differ by page and head."""
    from qwen_triton_b200.ops import kernels
    gen = torch.Generator().manual_seed(seed)
    values = [(torch.randn((pages, kv_heads, PAGE, dim), generator=gen) * 90).clamp(-448, 448).to(E4M3) for _ in range(2)]
    scales = [torch.exp2(torch.randint(-9, -9 + spread, (pages, kv_heads), generator=gen).float()) for _ in range(2)]
    return kernels.Cache8(*(t.cuda() for t in (*values, *scales)))


def _held(cache):
    """(k, v) in float64 on the host."""
    return tuple(values.view(torch.uint8).cpu().view(E4M3).double() * scales.cpu().double()[..., None, None] for values, scales in ((cache.k, cache.k_scale), (cache.v, cache.v_scale)))


def _table(counts, pages, seed, width=None):
    gen = torch.Generator().manual_seed(seed)
    order = torch.randperm(pages, generator=gen).tolist()
    width = width or max(1, max(counts))
    rows = []
    for count in counts:
        rows.append([order.pop() for _ in range(count)] + [0] * (width - count))
    return torch.tensor(rows, dtype=torch.int32)


def _ints(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def _close(out, want, bound):
    bound = bound + want.abs() * torch.finfo(out.dtype).eps / 2 * (1 + 2 ** -8) + 1e-30
    off = (out.double().cpu() - want).abs()
    assert bool((off <= bound).all()), f"{float((off / bound).max())} of the bound"


DIGITS = {BF16: 11, F32: 20}          # a weight is a half (11 digits), or two


def _decode(lengths, heads, kv_heads, dim, dtype, seed=0, ranges=None, spread=3, scale=None, cache=None):
    from qwen_triton_b200.ops import kernels
    counts = [-(-n // PAGE) for n in lengths]
    pages = sum(counts) + 2
    cache = cache or _filled(pages, kv_heads, dim, seed, spread)
    table = _table(counts, pages, seed)
    gen = torch.Generator().manual_seed(seed + 1)
    q = torch.randn((len(lengths), heads, dim), generator=gen).to(dtype)
    plan = kernels.decode8_plan(len(lengths), num_heads=heads, num_kv_heads=kv_heads, head_dim=dim, dtype=dtype, max_context=max(lengths))
    if ranges is not None:
        plan = kernels.Decode8Plan(plan.q_shape, kv_heads, dtype, *ranges)
    out = torch.full_like(q, math.nan, device="cuda")
    scratch = [torch.full((n,), math.nan, device="cuda") for n in (plan.acc_elements, plan.ml_elements)]
    scale = dim ** -0.5 if scale is None else scale
    kernels.attention_decode_cache8(q.cuda(), cache, out, table.cuda(), _ints(lengths), scale, plan, *scratch)
    want, bound = plain.attention(q, *_held(cache), table, [1] * len(lengths), [n - 1 for n in lengths], scale, DIGITS[dtype])
    _close(out, want, bound)


@pytest.mark.parametrize("heads,kv_heads,dim", HEADS)
@pytest.mark.parametrize("dtype", [BF16, F32])
def test_decode_heads(heads, kv_heads, dim, dtype):
    _decode([700, 1, 64, 65, 0, 333], heads, kv_heads, dim, dtype)


@pytest.mark.parametrize("length", [1, 2, 15, 16, 17, 31, 32, 33, 63, 64, 65, 127, 128, 129, 255, 257, 1000, 5001])
def test_decode_lengths(length):
    _decode([length], 8, 2, 128, BF16, seed=length)
    _decode([length, 3], 4, 4, 64, F32, seed=length)


@pytest.mark.parametrize("ranges", [(1, 1000), (1, 1), (2, 6), (4, 3), (7, 2), (13, 1), (3, 1), (64, 5), (9, 2), (16, 1), (2, 6, False), (7, 2, False), (5, 1, False)])
@pytest.mark.parametrize("dtype", [BF16, F32])
def test_decode_in_ranges(ranges, dtype):
    """Any cut gives the result: ranges that are empty, a last one that takes many pages, sequences without keys."""
    _decode([800, 0, 1, 129, 640, 64], 8, 2, 128, dtype, ranges=ranges)
    _decode([130, 64, 0], 12, 1, 48, dtype, ranges=ranges)


def test_decode_of_many_sequences():
    _decode([(37 * i) % 500 for i in range(70)], 16, 8, 128, BF16)


@pytest.mark.parametrize("dtype", [BF16, F32])
def test_decode_with_scales_far_apart(dtype):
    """Pages whose values differ by up to 2^30 in size, scores up to the hundreds, and a scale of the scores that is negative."""
    _decode([900, 65], 8, 2, 128, dtype, spread=30, scale=1e-3)
    _decode([900, 65], 8, 2, 64, dtype, spread=4, scale=2.0)
    _decode([200, 65], 8, 2, 64, dtype, scale=-0.1)


def test_what_lies_behind_the_last_key_is_not_looked_at():
    """NaN in the places behind a sequence's end, in pages that it does not list, and in what its page list says behind its last page."""
    from qwen_triton_b200.ops import kernels
    lengths = [70, 64, 1]
    for dtype in (BF16, F32):
        cache = _filled(6, 2, 64, 11)
        table = torch.tensor([[3, 1, -7], [0, 10 ** 9, 5], [4, 2, 2]], dtype=torch.int32)
        for t in (cache.k, cache.v):
            raw = t.view(torch.uint8)
            raw[1, :, 6:] = 0x7f
            raw[4, :, 1:] = 0xff
            raw[2] = raw[5] = 0x7f
        for t in (cache.k_scale, cache.v_scale):
            t[2] = t[5] = math.nan
        q = torch.randn((3, 4, 64), generator=torch.Generator().manual_seed(2)).to(dtype)
        want, bound = plain.attention(q, *_held(cache), table, [1] * 3, [n - 1 for n in lengths], 0.125, DIGITS[dtype])
        for ranges in ((1, 9), (2, 1), (3, 1), (12, 1)):
            plan = kernels.Decode8Plan((3, 4, 64), 2, dtype, *ranges)
            out = torch.full_like(q, math.nan, device="cuda")
            scratch = [torch.full((n,), math.nan, device="cuda") for n in (plan.acc_elements, plan.ml_elements)]
            kernels.attention_decode_cache8(q.cuda(), cache, out, table.cuda(), _ints(lengths), 0.125, plan, *scratch)
            _close(out, want, bound)
        out = torch.full_like(q, math.nan, device="cuda")
        for impl in ("tc", "mma") if dtype == BF16 else ("mma",):
            kernels.attention_prefill_cache8(q.cuda(), cache, out, table.cuda(), _ints([0, 1, 2, 3]), _ints([n - 1 for n in lengths]), 1, 0.125, impl)
            _close(out, *plain.attention(q, *_held(cache), table, [1] * 3, [n - 1 for n in lengths], 0.125, DIGITS[dtype], impl == "tc"))


@pytest.mark.parametrize("ranges", [(2, 10 ** 9), (8, 2 ** 31 - 1), (3, 2 ** 30, False), (64, 2 ** 31 - 1, False)])
def test_ranges_of_more_pages_than_there_are(ranges):
    """The first range has every key, whatever its size in pages times ranges comes to."""
    _decode([70, 200, 1], 4, 2, 64, BF16, 3, ranges)


def test_a_nan_that_is_seen_is_handed_on():
    from qwen_triton_b200.ops import kernels
    cache = _filled(3, 1, 64, 12)
    cache.k.view(torch.uint8)[1, 0, 5, 3] = 0x7f
    q = torch.ones((2, 1, 64), dtype=BF16, device="cuda")
    out = torch.empty_like(q)
    for ranges in ((1, 9), (2, 1), (9, 1)):
        plan = kernels.Decode8Plan((2, 1, 64), 1, BF16, *ranges)
        scratch = [torch.empty(n, device="cuda") for n in (plan.acc_elements, plan.ml_elements)]
        kernels.attention_decode_cache8(q, cache, out, _ints([[0, 1], [2, 0]]), _ints([100, 64]), 0.1, plan, *scratch)
        assert bool(out[0].isnan().all()) and bool(out[1].isfinite().all())


def _prompt(counts, past, heads, kv_heads, dim, dtype, seed=0, scale=None, spread=3, impl=None, ranges=None):
    from qwen_triton_b200.ops import kernels
    pages_of = [-(-(n + p) // PAGE) for n, p in zip(counts, past)]
    pages = sum(pages_of) + 1
    cache = _filled(pages, kv_heads, dim, seed, spread)
    table = _table(pages_of, pages, seed)
    q = torch.randn((sum(counts), heads, dim), generator=torch.Generator().manual_seed(seed + 1)).to(dtype)
    scale = dim ** -0.5 if scale is None else scale
    starts = [sum(counts[:i]) for i in range(len(counts) + 1)]
    want = {}
    for form in (impl,) if impl else ("tc", "mma") if dtype == BF16 and dim <= 128 and scale > 0 else ("mma",):
        out = torch.full_like(q, math.nan, device="cuda")
        kernels.attention_prefill_cache8(q.cuda(), cache, out, table.cuda(), _ints(starts), _ints(past), max(counts), scale, form, ranges)
        _close(out, *plain.attention(q, *_held(cache), table, counts, past, scale, DIGITS[dtype], form == "tc"))
    kernels.check_status()


@pytest.mark.parametrize("heads,kv_heads,dim", HEADS)
@pytest.mark.parametrize("dtype", [BF16, F32])
def test_prompt_heads(heads, kv_heads, dim, dtype):
    _prompt([70, 1, 33], [0, 100, 64], heads, kv_heads, dim, dtype)


@pytest.mark.parametrize("count,past", [(1, 0), (2, 0), (63, 0), (64, 0), (65, 0), (127, 1), (128, 0), (129, 63), (200, 1000), (300, 7), (64, 64), (513, 129), (5, 2000)])
@pytest.mark.parametrize("heads,kv_heads,dim", [(8, 2, 128), (3, 1, 64), (2, 2, 128)])
def test_prompt_lengths(count, past, heads, kv_heads, dim):
    _prompt([count], [past], heads, kv_heads, dim, BF16, seed=count)


def test_prompts_of_many_sequences():
    """Prompts of all lengths in one call, one of them without tokens."""
    _prompt([1, 130, 0, 64, 257, 12, 300], [0, 5, 64, 0, 700, 129, 0], 8, 2, 128, BF16)
    _prompt([1, 130, 0, 64, 257, 12, 300], [0, 5, 64, 0, 700, 129, 0], 6, 2, 64, BF16)
    _prompt([1, 130, 0, 64], [0, 5, 64, 0], 6, 2, 64, F32)


@pytest.mark.parametrize("ranges", [1, 2, 3, 7, 8])
@pytest.mark.parametrize("dtype", [BF16, F32])
def test_prompts_in_ranges(ranges, dtype):
    """A tile's keys by clusters of every size, more blocks than pages among them, sequences without tokens."""
    _prompt([3, 20, 0, 1, 70], [0, 700, 64, 5, 63], 8, 2, 128, dtype, ranges=ranges)
    _prompt([3, 20, 0, 1, 70], [0, 700, 64, 5, 63], 3, 1, 48, dtype, ranges=ranges)
    _prompt([150, 0, 300], [1500, 64, 0], 6, 2, 64, dtype, ranges=ranges)
    _prompt([200, 1], [900, 2100], 4, 4, 112, dtype, ranges=ranges)


@pytest.mark.parametrize("heads,kv_heads,dim", [(8, 2, 128), (4, 2, 64), (4, 2, 48)])
def test_prompt_with_scales_far_apart(heads, kv_heads, dim):
    _prompt([150, 70], [300, 0], heads, kv_heads, dim, BF16, spread=30, scale=1e-3)
    _prompt([150, 70], [300, 0], heads, kv_heads, dim, BF16, spread=4, scale=2.0)
    _prompt([150, 70], [300, 0], heads, kv_heads, dim, BF16, scale=-0.1)
    _prompt([150, 70], [300, 0], heads, kv_heads, dim, BF16, scale=0.0)


@pytest.mark.parametrize("dim", [64, 128])
def test_prompt_queries_of_all_sizes(dim):
    """Rows of zeros, of the smallest and the largest numbers, elements far below the row's largest; a row with an infinity is NaN, the others are as without it."""
    from qwen_triton_b200.ops import kernels
    counts, past = [90], [70]
    cache, table = _filled(4, 1, dim, 3), torch.tensor([[2, 0, 1]], dtype=torch.int32)
    gen = torch.Generator().manual_seed(9)
    q = torch.randn((90, 2, dim), generator=gen) * torch.exp2(torch.randint(-14, 1, (90, 2, dim), generator=gen).float())
    q[3] = 0
    q[5] *= 2.0 ** -100
    q[7] *= 2.0 ** 10
    q = q.to(BF16)
    want = {impl: plain.attention(q, *_held(cache), table, counts, past, dim ** -0.5, DIGITS[BF16], impl == "tc") for impl in ("tc", "mma")}
    q[11, 1, 5] = math.inf
    for impl in ("tc", "mma"):
        out = torch.full_like(q, math.nan, device="cuda")
        kernels.attention_prefill_cache8(q.cuda(), cache, out, table.cuda(), _ints([0, 90]), _ints(past), 90, dim ** -0.5, impl)
        assert bool(out[11, 1].isnan().all())
        out[11, 1] = 0
        for part in want[impl]:
            part[11, 1] = 0
        _close(out, *want[impl])
    kernels.check_status()


# ----------------------------------------------------------------------------- the write
def _write_inputs(counts, past, heads, kv_heads, dim, dtype, planes, seed):
    from qwen_triton_b200.ops import kernels
    gen = torch.Generator().manual_seed(seed)
    pages_of = [max(1, -(-(n + p) // PAGE)) for n, p in zip(counts, past)]
    pages = sum(pages_of) + 2
    cache = _filled(pages, kv_heads, dim, seed)
    table = _table(pages_of, pages, seed)
    tokens = sum(counts)
    qkv = torch.randn((planes, tokens, (heads + 2 * kv_heads) * dim), generator=gen).to(dtype)
    cos_sin = torch.randn((max(n + p for n, p in zip(counts, past)) + 1, dim), generator=gen)
    weights = [1 + 0.2 * torch.randn(dim, generator=gen) for _ in range(2)]
    starts = [sum(counts[:i]) for i in range(len(counts) + 1)]
    position = torch.tensor([p + j for n, p in zip(counts, past) for j in range(n)], dtype=torch.long)
    return cache, table, qkv, cos_sin, weights, starts, position, gen


def _bits(cache):
    return [t.view(torch.uint8).cpu().clone() for t in (cache.k, cache.v)] + [t.cpu().clone() for t in (cache.k_scale, cache.v_scale)]


def _check_write(counts, past, heads, kv_heads, dim, dtype=BF16, out_dtype=None, planes=1, norm=True, rotate=True, interleaved=False, rotary=None, seed=0):
    from qwen_triton_b200.ops import kernels
    cache, table, qkv, cos_sin, weights, starts, position, _ = _write_inputs(counts, past, heads, kv_heads, dim, dtype, planes, seed)
    cos_sin = cos_sin[:, :rotary].contiguous() if rotary else cos_sin
    q = torch.full((sum(counts), heads, dim), math.nan, dtype=out_dtype or dtype, device="cuda")
    want = [(t.view(torch.uint8).cpu().view(E4M3).double(), s.cpu().double()) for t, s in ((cache.k, cache.k_scale), (cache.v, cache.v_scale))]
    kernels.qkv_write_cache8(kernels.GemmOut(qkv.cuda()), q, cache, _ints(starts), _ints(past), table.cuda(), max(counts), weights[0].cuda() if norm else None,
                             weights[1].cuda() if norm else None, 1e-6, cos_sin.cuda() if rotate else None, interleaved=interleaved)
    x = qkv.double().sum(0).view(-1, heads + 2 * kv_heads, dim)
    parts = [plain.treated(part, weight if norm else None, 1e-6, cos_sin if rotate and weight is not None else None, position, interleaved)
             for part, weight in ((x[:, :heads], weights[0]), (x[:, heads:heads + kv_heads], weights[1]))]
    # two products and an addition of numbers that carry the norm's (d + 4 roundings), the planes' sums and the weight's roundings
    size = 2 * parts[0].abs().amax() + 1e-30
    _close(q, parts[0], size * (dim + 16) * 2.0 ** -24)
    for (values, scales), rows, got, got_scale in zip(want, (parts[1], x[:, heads + kv_heads:]), (cache.k, cache.v), (cache.k_scale, cache.v_scale)):
        plain.write(values, scales, rows, table, starts, past)
        assert torch.equal(got_scale.cpu().double(), scales)
        got = got.view(torch.uint8).cpu().view(E4M3).double()
        # a number next to a border between two e4m3 numbers may fall on either side: one step, and rarely
        differ = got != values
        step = torch.exp2((torch.frexp(values)[1] - 1).clamp(min=-6).double() - 3)
        assert bool(((got - values).abs() <= step)[differ].all()) and int(differ.sum()) <= 2 + values.numel() * 2e-5


@pytest.mark.parametrize("heads,kv_heads,dim", HEADS)
def test_write_heads(heads, kv_heads, dim):
    _check_write([70, 1, 5], [0, 63, 120], heads, kv_heads, dim)


@pytest.mark.parametrize("counts,past", [([1], [0]), ([1] * 9, [0, 1, 62, 63, 64, 65, 500, 127, 128]), ([64], [0]), ([65], [0]), ([200], [1]), ([64, 64], [64, 32]),
                                         ([300, 0, 1, 17], [7, 64, 64, 47])])
@pytest.mark.parametrize("dtype,planes", [(BF16, 1), (F32, 1), (F32, 3)])
def test_write_lengths(counts, past, dtype, planes):
    _check_write(counts, past, 4, 2, 128, dtype, BF16, planes)


@pytest.mark.parametrize("norm,rotate,interleaved,rotary", [(False, False, False, None), (True, False, False, None), (False, True, False, None), (True, True, True, None),
                                                            (True, True, False, 32), (True, True, True, 48)])
@pytest.mark.parametrize("counts,past", [([1, 1, 1], [5, 64, 0]), ([80, 3], [0, 62])])
def test_write_treatments(norm, rotate, interleaved, rotary, counts, past):
    _check_write(counts, past, 4, 2, 64, F32, F32, 1, norm, rotate, interleaved, rotary)
    _check_write(counts, past, 4, 2, 64, BF16, BF16, 1, norm, rotate, interleaved, rotary)


@pytest.mark.parametrize("pieces", [(100,), (1,) * 100, (30, 40, 30), (64, 36), (63, 1, 1, 35)])
def test_a_page_written_in_pieces_is_as_if_written_at_once(pieces):
    """Scales are those of all numbers in a page; numbers differ only where a smaller scale held one below 2^-6 of the larger."""
    from qwen_triton_b200.ops import kernels
    cache, table, qkv, _, _, _, _, gen = _write_inputs([100], [0], 2, 1, 64, F32, 1, 5)
    qkv *= torch.exp2(torch.linspace(0, 9, 100))[None, :, None]          # every few tokens raise the scale
    at = 0
    for n in pieces:
        q = torch.empty((n, 2, 64), device="cuda")
        kernels.qkv_write_cache8(kernels.GemmOut(qkv[:, at:at + n].contiguous().cuda()), q, cache, _ints([0, n]), _ints([at]), table.cuda(), n, None, None, 0.0, None)
        at += n
    whole = qkv[0].double().view(100, 4, 64)
    for heads, got, got_scale in ((whole[:, 2:3], cache.k, cache.k_scale), (whole[:, 3:], cache.v, cache.v_scale)):
        got = got.view(torch.uint8).cpu().view(E4M3).double()
        for page in range(2):
            rows = heads[page * 64:(page + 1) * 64, 0]
            p = int(table[0, page])
            scale = 2.0 ** plain.power_for(float(rows.abs().max()))
            assert float(got_scale[p, 0]) == scale
            want = plain.as_e4m3(rows / scale)
            held = got[p, 0, :len(rows)]
            small = want.abs() <= 2.0 ** -6
            assert torch.equal(held[~small], want[~small])
            # each of the at most nine steps that brought it down rounded to a multiple of 2^-9
            assert bool(((held - rows / scale).abs() <= 10 * 2.0 ** -10)[small].all())


def test_write_leaves_the_rest_alone():
    """The bytes behind the last token, the pages of others, and a call without tokens."""
    from qwen_triton_b200.ops import kernels
    cache, table, qkv, cos_sin, weights, starts, _, _ = _write_inputs([3, 70], [5, 10], 4, 2, 64, BF16, 1, 6)
    before = _bits(cache)
    q = torch.empty((73, 4, 64), dtype=BF16, device="cuda")
    args = (q, cache, _ints(starts), _ints([5, 10]), table.cuda(), 70, weights[0].cuda(), weights[1].cuda(), 1e-6, cos_sin.cuda())
    kernels.qkv_write_cache8(kernels.GemmOut(qkv.cuda()), *args)
    after = _bits(cache)
    touched = {int(table[0, 0]): 8, int(table[1, 0]): 64, int(table[1, 1]): 16}
    for old, new in zip(before[:2], after[:2]):
        for page in range(old.shape[0]):
            assert torch.equal(old[page, :, touched.get(page, 0):], new[page, :, touched.get(page, 0):])
    for old, new in zip(before[2:], after[2:]):
        others = [page for page in range(old.shape[0]) if page not in touched]
        assert torch.equal(old[others], new[others])
    # the same call once more changes nothing
    kernels.qkv_write_cache8(kernels.GemmOut(qkv.cuda()), *args)
    assert all(torch.equal(a, b) for a, b in zip(after, _bits(cache)))
    kernels.qkv_write_cache8(kernels.GemmOut(qkv[:, :0].contiguous().cuda()), q[:0], cache, _ints([0, 0, 0]), _ints([5, 10]), table.cuda(), 0, None, None, 0.0, None)
    assert all(torch.equal(a, b) for a, b in zip(after, _bits(cache)))


@pytest.mark.parametrize("dtype", [BF16, F32])
def test_numbers_at_the_ends_of_the_range(dtype):
    """Zeros take the smallest scale, numbers beyond the largest one end there, infinities and NaN are held as NaN and do not move the scale."""
    from qwen_triton_b200.ops import kernels
    cache = _filled(2, 1, 16, 7)
    qkv = torch.ones((1, 6, 48))
    qkv[0, :, 16:] = 0
    qkv[0, 1, 16] = 2.0 ** -30
    rows = [(qkv[:, :2], 2.0 ** -38)]
    big = torch.ones((1, 2, 48)) * 1e20
    infinite = torch.ones((1, 3, 48)) * 3.5
    infinite[0, 1, 20], infinite[0, 1, 40], infinite[0, 2, 47] = math.inf, -math.inf, math.nan
    for x, scale in (*rows, (big, 2.0 ** 40), (infinite, 2.0 ** -7)):
        x = x.to(dtype)
        n = x.shape[1]
        q = torch.empty((n, 1, 16), dtype=dtype, device="cuda")
        kernels.qkv_write_cache8(kernels.GemmOut(x.contiguous().cuda()), q, cache, _ints([0, n]), _ints([0]), _ints([[1]]), n, None, None, 0.0, None)
        for part, got, got_scale in ((x[0, :, 16:32], cache.k, cache.k_scale), (x[0, :, 32:], cache.v, cache.v_scale)):
            finite = part.double()[part.isfinite()].abs().max()
            assert float(got_scale[1, 0]) == 2.0 ** plain.power_for(float(finite))
            want = plain.as_e4m3(part.double() / float(got_scale[1, 0]))
            held = got.view(torch.uint8).cpu().view(E4M3).double()[1, 0, :n]
            assert torch.equal(held.nan_to_num(1e9), want.nan_to_num(1e9))
    assert float(cache.k_scale[1, 0]) == 2.0 ** -7


# ----------------------------------------------------------------------------- together
@pytest.mark.parametrize("dtype", [BF16, F32])
def test_a_prompt_and_steps_behind_it(dtype):
    """Two prompts in two pieces each, then single tokens across a page's end, captured and replayed: as attention over what the cache then holds, and near to attention
    over keys and values that were never brought to 8 bits."""
    from qwen_triton_b200.ops import kernels
    heads, kv_heads, dim, width = 8, 2, 64, 4
    gen = torch.Generator().manual_seed(3)
    cache = kernels.cache8(9, kv_heads, dim, "cuda")
    table = torch.tensor([[3, 1, 7, 0], [2, 8, 4, 0]], dtype=torch.int32).cuda()
    angle = torch.arange(256)[:, None] * 1e4 ** (-torch.arange(0, dim, 2) / dim)
    cos_sin = torch.cat((angle.cos(), angle.sin()), 1)
    weights = [1 + 0.1 * torch.randn(dim, generator=gen) for _ in range(2)]
    past, sequences = [0, 0], [[], []]

    def project(counts):
        rows = torch.randn((sum(counts), (heads + 2 * kv_heads) * dim), generator=gen).to(dtype)
        at = 0
        for i, n in enumerate(counts):
            sequences[i].append(rows[at:at + n])
            at += n
        return rows

    def check(out, counts, q):
        want, bound = plain.attention(q.cpu(), *_held(cache), table.cpu(), counts, past, dim ** -0.5, DIGITS[dtype], dtype == BF16)
        _close(out, want, bound)
        # without 8 bits: a key's numbers are off by 2^-4 of themselves at most, a value's too
        at = 0
        for i, n in enumerate(counts):
            x = torch.cat(sequences[i]).double().view(-1, heads + 2 * kv_heads, dim)
            place = torch.arange(len(x))
            k = plain.treated(x[:, heads:heads + kv_heads], weights[1], 1e-6, cos_sin, place)
            v = x[:, heads + kv_heads:]
            for h in range(heads):
                s = q.double().cpu()[at:at + n, h] @ k[:, h // 4].T * dim ** -0.5
                s = s.masked_fill(torch.arange(len(x))[None] > past[i] + torch.arange(n)[:, None], -math.inf)
                full = torch.softmax(s, 1) @ v[:, h // 4]
                off = (out.double().cpu()[at:at + n, h] - full).norm() / full.norm()
                assert float(off) < 0.1
            at += n

    for counts in ([50, 70], [30, 90]):
        qkv = project(counts)
        q = torch.empty((sum(counts), heads, dim), dtype=dtype, device="cuda")
        out = torch.empty_like(q)
        starts = _ints([0, counts[0], sum(counts)])
        kernels.qkv_write_cache8(kernels.GemmOut(qkv[None].cuda()), q, cache, starts, _ints(past), table, max(counts), weights[0].cuda(), weights[1].cuda(), 1e-6, cos_sin.cuda())
        kernels.attention_prefill_cache8(q, cache, out, table, starts, _ints(past), max(counts), dim ** -0.5)
        check(out, counts, q)
        past = [p + n for p, n in zip(past, counts)]
    plan = kernels.decode8_plan(2, num_heads=heads, num_kv_heads=kv_heads, head_dim=dim, dtype=dtype, max_context=width * PAGE)
    scratch = [torch.empty(n, device="cuda") for n in (plan.acc_elements, plan.ml_elements)]
    q = torch.empty((2, heads, dim), dtype=dtype, device="cuda")
    out, qkv_in, past_in, len_in = torch.empty_like(q), torch.zeros((1, 2, (heads + 2 * kv_heads) * dim), dtype=dtype, device="cuda"), _ints(past), _ints([p + 1 for p in past])
    fixed = (weights[0].cuda(), weights[1].cuda(), 1e-6, cos_sin.cuda())
    starts = _ints([0, 1, 2])

    def step():
        kernels.qkv_write_cache8(kernels.GemmOut(qkv_in), q, cache, starts, past_in, table, 1, *fixed)
        kernels.attention_decode_cache8(q, cache, out, table, len_in, dim ** -0.5, plan, *scratch)

    graph = None
    for turn in range(50):
        qkv_in.copy_(project([1, 1])[None])
        past_in.copy_(_ints(past))
        len_in.copy_(_ints([p + 1 for p in past]))
        if turn == 1:
            torch.cuda.synchronize()
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph):
                step()
        if graph is None:
            step()
        else:
            graph.replay()
        torch.cuda.synchronize()
        if turn % 7 == 0 or turn > 46:
            check(out, [1, 1], q)
        past = [p + 1 for p in past]


def test_on_another_stream():
    from qwen_triton_b200.ops import kernels
    stream = torch.cuda.Stream()
    with torch.cuda.stream(stream):
        _decode([300, 64], 8, 2, 128, BF16)
        _prompt([100, 64], [0, 64], 8, 2, 128, BF16)
    stream.synchronize()


def test_pages_beyond_32_bits():
    """Pages that begin more than 2^31 and 2^32 bytes into a cache, listed also twice: the results are those of the same contents in a small cache, bit by bit."""
    from qwen_triton_b200.ops import kernels
    heads, kv_heads, dim = 16, 8, 128
    far = 66000                                            # pages of 64 KB: 4.3 GB each of keys and values
    places = [far - 1, 33000, 3, 65536, 32768]             # of the small cache's pages
    small, large = kernels.cache8(5, kv_heads, dim, "cuda"), kernels.cache8(far, kv_heads, dim, "cuda")
    table = torch.tensor([[0, 1, 2, 0], [3, 4, 4, 4]], dtype=torch.int32)
    moved = torch.tensor(places, dtype=torch.int32)[table.long()]
    gen = torch.Generator().manual_seed(5)
    qkv = torch.randn((1, 300, (heads + 2 * kv_heads) * dim), generator=gen).to(BF16).cuda()
    starts, none = _ints([0, 180, 300]), _ints([0, 0])
    got = []
    for cache, pages in ((small, table.cuda()), (large, moved.cuda())):
        q = torch.empty((300, heads, dim), dtype=BF16, device="cuda")
        kernels.qkv_write_cache8(kernels.GemmOut(qkv), q, cache, starts, none, pages, 180, None, None, 1e-6, None)
        one = kernels.GemmOut(qkv[:, :2].contiguous())
        kernels.qkv_write_cache8(one, q[:2], cache, _ints([0, 1, 2]), _ints([180, 120]), pages, 1, None, None, 1e-6, None)
        outs = [q]
        for impl, ranges in (("tc", 1), ("tc", 2), ("mma", 1), ("mma", 3)):
            outs.append(torch.empty_like(q))
            kernels.attention_prefill_cache8(q, cache, outs[-1], pages, starts, _ints([70, 100]), 180, 0.1, impl, ranges)
        for ranges in ((1, 4), (4, 1), (2, 2, False)):
            plan = kernels.Decode8Plan((2, heads, dim), kv_heads, BF16, *ranges)
            scratch = [torch.empty(n, device="cuda") for n in (plan.acc_elements, plan.ml_elements)]
            outs.append(torch.empty((2, heads, dim), dtype=BF16, device="cuda"))
            kernels.attention_decode_cache8(q[:2].contiguous(), cache, outs[-1], pages, _ints([250, 256]), 0.1, plan, *scratch)
        got.append(outs)
    for a, b in zip(*got):
        assert bool(a.isfinite().all()) and torch.equal(a, b)
    index = torch.tensor(places, device="cuda")
    for a, b in ((small.k, large.k), (small.v, large.v)):
        assert torch.equal(a.view(torch.uint8), b.view(torch.uint8)[index])
    assert torch.equal(small.k_scale, large.k_scale[index]) and torch.equal(small.v_scale, large.v_scale[index])


def test_two_graphs_that_share_scratch():
    """Captured calls of other lengths over one cache and one scratch, replayed in turns: each replay's results are its launched call's."""
    from qwen_triton_b200.ops import kernels
    cache = _filled(20, 2, 64, 6)
    tables, lengths = _table([9, 7], 20, 1).cuda(), ([560, 430], [3, 448])
    q = torch.randn((2, 4, 64), generator=torch.Generator().manual_seed(2)).to(BF16).cuda()
    plan = kernels.Decode8Plan((2, 4, 64), 2, BF16, 9, 1)
    scratch = [torch.empty(n, device="cuda") for n in (plan.acc_elements, plan.ml_elements)]
    lens, outs, wants, graphs = [_ints(n) for n in lengths], [], [], []
    for n in lens:
        want, out, graph = torch.empty_like(q), torch.empty_like(q), torch.cuda.CUDAGraph()
        kernels.attention_decode_cache8(q, cache, want, tables, n, 0.1, plan, *scratch)
        torch.cuda.synchronize()
        with torch.cuda.graph(graph):
            kernels.attention_decode_cache8(q, cache, out, tables, n, 0.1, plan, *scratch)
        outs.append(out), wants.append(want), graphs.append(graph)
    for turn in range(6):
        outs[turn % 2].fill_(math.nan)
        graphs[turn % 2].replay()
        assert torch.equal(outs[turn % 2], wants[turn % 2])


def test_launches_are_counted():
    from qwen_triton_b200.ops import kernels
    from test_gpu_launch_counts import kernels_of
    cache, table = kernels.cache8(20, 2, 64, "cuda"), _table([9, 7], 20, 1).cuda()
    q = torch.ones((2, 4, 64), dtype=BF16, device="cuda")
    out, lens, starts, past = torch.empty_like(q), _ints([500, 400]), _ints([0, 1, 2]), _ints([499, 399])
    for ranges, launches in (((1, 9), 1), ((4, 3), 1), ((4, 3, False), 2), ((9, 1), 2)):
        plan = kernels.Decode8Plan((2, 4, 64), 2, BF16, *ranges)
        scratch = [torch.empty(n, device="cuda") for n in (plan.acc_elements, plan.ml_elements)]
        assert kernels_of(lambda: kernels.attention_decode_cache8(q, cache, out, table, lens, 0.1, plan, *scratch)) == (launches, launches)
    for impl, ranges in (("tc", 1), ("tc", 3), ("mma", 1), ("mma", 3)):
        assert kernels_of(lambda: kernels.attention_prefill_cache8(q, cache, out, table, starts, past, 1, 0.1, impl, ranges)) == (1, 1)
    qkv = kernels.GemmOut(torch.ones((1, 2, 512), dtype=BF16, device="cuda"))
    for most in (1, 2):
        assert kernels_of(lambda: kernels.qkv_write_cache8(qkv, q, cache, starts, past, table, most, None, None, 1e-6, None)) == (1, 1)


def test_refusals():
    from qwen_triton_b200.ops import kernels
    Error = kernels.KernelError
    cache = _filled(4, 2, 64, 1)
    with pytest.raises(Error, match="keys"):
        kernels.cache8(4, 2, 72, "cuda")
    with pytest.raises(Error, match="keys"):
        kernels.cache8(4, 2, 272, "cuda")
    with pytest.raises(Error, match="v must"):
        kernels.Cache8(cache.k, cache.v[:3], cache.k_scale, cache.v_scale)
    with pytest.raises(Error, match="k_scale"):
        kernels.Cache8(cache.k, cache.v, cache.k_scale[:, :1].contiguous(), cache.v_scale)
    with pytest.raises(Error, match="must be torch.float8"):
        kernels.Cache8(cache.k.view(torch.uint8), cache.v, cache.k_scale, cache.v_scale)
    q = torch.zeros((2, 4, 64), dtype=BF16, device="cuda")
    out, table, lens = torch.empty_like(q), _ints([[0, 1], [2, 3]]), _ints([100, 3])
    plan = kernels.Decode8Plan((2, 4, 64), 2, BF16, 9, 1)
    acc, ml = (torch.empty(n, device="cuda") for n in (plan.acc_elements, plan.ml_elements))
    decode = kernels.attention_decode_cache8
    decode(q, cache, out, table, lens, 0.1, plan, acc, ml)
    with pytest.raises(Error, match="part_acc"):
        decode(q, cache, out, table, lens, 0.1, plan)
    with pytest.raises(Error, match="part_ml"):
        decode(q, cache, out, table, lens, 0.1, plan, acc, ml[:-1])
    with pytest.raises(Error, match="65 ranges"):
        decode(q, cache, out, table, lens, 0.1, kernels.Decode8Plan((2, 4, 64), 2, BF16, 65, 1), acc, ml)
    with pytest.raises(Error, match="9 ranges of"):
        decode(q, cache, out, table, lens, 0.1, kernels.Decode8Plan((2, 4, 64), 2, BF16, 9, 2 ** 31), acc, ml)
    with pytest.raises(Error, match="plan"):
        decode(q[:1], cache, out[:1], table[:1], lens[:1], 0.1, plan, acc, ml)
    with pytest.raises(Error, match="out must"):
        decode(q, cache, out.float(), table, lens, 0.1, plan, acc, ml)
    with pytest.raises(Error, match="queries"):
        decode(q[:, :3].contiguous(), cache, out, table, lens, 0.1, plan, acc, ml)
    with pytest.raises(Error, match="neither"):
        decode(q.half(), cache, out.half(), table, lens, 0.1, plan, acc, ml)
    with pytest.raises(Error, match="block table"):
        decode(q, cache, out, table[:1], lens, 0.1, plan, acc, ml)
    with pytest.raises(Error, match="seq_len"):
        decode(q, cache, out, table, lens.long(), 0.1, plan, acc, ml)
    with pytest.raises(Error, match="CUDA"):
        decode(q.cpu(), cache, out, table, lens, 0.1, plan, acc, ml)
    prefill = kernels.attention_prefill_cache8
    with pytest.raises(Error, match="max_q_len"):
        prefill(q, cache, out, table, _ints([0, 1, 2]), _ints([0, 0]), 3, 0.1)
    with pytest.raises(Error, match="seq_start"):
        prefill(q, cache, out, table, _ints([0, 1]), _ints([0, 0]), 1, 0.1)
    for impl, scale in (("other", 0.1), ("tc", -0.1)):
        with pytest.raises(Error, match="impl"):
            prefill(q, cache, out, table, _ints([0, 1, 2]), _ints([0, 0]), 1, scale, impl)
    for impl, ranges in (("mma", 9), ("mma", 0), ("tc", 9)):
        with pytest.raises(Error, match="ranges"):
            prefill(q, cache, out, table, _ints([0, 1, 2]), _ints([0, 0]), 1, 0.1, impl, ranges)
    with pytest.raises(Error, match="impl"):
        prefill(q.float(), cache, out.float(), table, _ints([0, 1, 2]), _ints([0, 0]), 1, 0.1, "tc")
    qkv = kernels.GemmOut(torch.zeros((1, 2, 512), dtype=BF16, device="cuda"))
    write = kernels.qkv_write_cache8
    write(qkv, q, cache, _ints([0, 1, 2]), _ints([0, 0]), table, 1, None, None, 0.0, None)
    with pytest.raises(Error, match="projection"):
        write(kernels.GemmOut(qkv.tensor[..., :448].contiguous()), q, cache, _ints([0, 1, 2]), _ints([0, 0]), table, 1, None, None, 0.0, None)
    with pytest.raises(Error, match="rotary"):
        write(qkv, q, cache, _ints([0, 1, 2]), _ints([0, 0]), table, 1, None, None, 0.0, torch.zeros((9, 66), device="cuda"))
    with pytest.raises(Error, match="q_weight"):
        write(qkv, q, cache, _ints([0, 1, 2]), _ints([0, 0]), table, 1, torch.ones(32, device="cuda"), None, 0.0, None)
