"""Attention over an 8-bit cache where single numbers decide: weights far below the largest one, and values that are not numbers."""
import math

import pytest
import torch

import plain_8bit as plain

pytestmark = pytest.mark.gpu
E4M3 = torch.float8_e4m3fn
PAGE = 64
BF16, F32 = torch.bfloat16, torch.float32
# What a weight may be off by, relative to itself, and relative to the largest of p_j s_v[j].  A half has 11 binary digits, 2^-12 at most; it ends at 2^-24, off by 2^-25 at
# most, and weights are held times 2^11 (the largest, whose reference may lag by 2^4, at most 2^15).  Float calls hold the remainder times 2^11 as another half: 2^-24, and 2^-11 of that.
OF_ITSELF, OF_LARGEST = {BF16: 2.0 ** -12, F32: 2.0 ** -23}, {BF16: 2.0 ** -36, F32: 2.0 ** -47}


def _ints(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def _cache(k8, v8, k_scale, v_scale):
    """Numbers [tokens, d] of one kv head, a multiple of 64 of them, as pages in order."""
    from qwen_triton_b200.ops import kernels
    k8, v8 = (t.float().to(E4M3).view(-1, 1, PAGE, t.shape[1]).cuda() for t in (k8, v8))
    return kernels.Cache8(k8, v8, k_scale.float().view(-1, 1).cuda(), v_scale.float().view(-1, 1).cuda())


def _expected(score, v8, v_scale, dtype):
    """(out, bound) of one query with these scores.  Here a query has one element that is not zero, so that a score's sum is exact; its scaling and the exponential are off by
    2^-21 of the score and 2^-21, which meet a result twice; sums over the keys by 2^-23 an addition, at most 200 in turn for a range and the joins, the others within an
    instruction of eight keys."""
    p = torch.softmax(score, 0)
    scale = v_scale.double().repeat_interleave(PAGE)[:, None]
    sizes = (v8.double() * scale).abs()
    relative = OF_ITSELF[dtype] + 2 * (float(score[score.isfinite()].abs().max()) + 1) * 2.0 ** -21 + (200 + len(score) / 8) * 2.0 ** -23
    lost = OF_LARGEST[dtype] * float((p[:, None] * scale).max()) * v8.double().abs().sum(0)
    out = p @ (v8.double() * scale)
    return out, relative * (p @ sizes) + lost + out.abs() * torch.finfo(dtype).eps / 2 * (1 + 2.0 ** -8)


def _far_below(length, dim, at, seed):
    """One key 18 nats above all others, whose value is 0 in every other element: these are sums of weights between e^-17 and e^-19."""
    gen = torch.Generator().manual_seed(seed)
    k8 = torch.randint(-8, 9, (length, dim), generator=gen).double()
    k8[:, 0] = torch.randint(-8, 9, (length,), generator=gen)
    k8[at, 0] = 288                                        # 18 under a scale of 2^-4
    v8 = torch.randint(8, 16, (length, dim), generator=gen).double() * 16
    v8[at, ::2] = 0
    pages = length // PAGE
    return k8, v8, torch.full((pages,), 2.0 ** -4), torch.exp2(torch.randint(-9, -6, (pages,), generator=gen).float())


def _beside_large_scale(length, dim, at, seed):
    """One page whose values are under a scale 2^20 times the others', and 0 in every other element: there the others alone are left."""
    k8, v8, k_scale, v_scale = _far_below(length, dim, at, seed)
    k8[at, 0] = 0
    v8[at // PAGE * PAGE:(at // PAGE + 1) * PAGE, ::2] = 0
    v_scale[:] = 2.0 ** -8
    v_scale[at // PAGE] = 2.0 ** 12
    return k8, v8, k_scale, v_scale


@pytest.mark.parametrize("kind", [_far_below, _beside_large_scale])
@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("dim,ranges", [(128, (1, 1000)), (64, (4, 32)), (128, (16, 8, False)), (256, (2, 64))])
@pytest.mark.parametrize("at", [3, 4000, 8190])
def test_decode_of_small_weights(kind, dtype, dim, ranges, at):
    from qwen_triton_b200.ops import kernels
    k8, v8, k_scale, v_scale = kind(8192, dim, at, dim + at)
    cache = _cache(k8, v8, k_scale, v_scale)
    q = torch.zeros((1, 2, dim), dtype=dtype)
    q[..., 0] = 1
    plan = kernels.Decode8Plan((1, 2, dim), 1, dtype, *ranges)
    out = torch.full_like(q, math.nan, device="cuda")
    scratch = [torch.full((n,), math.nan, device="cuda") for n in (plan.acc_elements, plan.ml_elements)]
    kernels.attention_decode_cache8(q.cuda(), cache, out, torch.arange(128, dtype=torch.int32)[None].cuda(), _ints([8192]), 1.0, plan, *scratch)
    want, bound = _expected(k8[:, 0] / 16, v8, v_scale, dtype)
    off = (out.double().cpu() - want).abs()
    assert bool((off <= bound).all()), f"{float((off / bound).max())} of the bound"


@pytest.mark.parametrize("kind", [_far_below, _beside_large_scale])
@pytest.mark.parametrize("impl,dtype,dim", [("mma", BF16, 128), ("mma", F32, 128), ("mma", F32, 256), ("mma", F32, 48), ("tc", BF16, 128), ("tc", BF16, 64), ("tc", BF16, 80)])
@pytest.mark.parametrize("at,ranges", [(3, 1), (4000, 1), (4000, 4), (8100, 3)])
def test_prompt_of_small_weights(kind, impl, dtype, dim, at, ranges):
    from qwen_triton_b200.ops import kernels
    k8, v8, k_scale, v_scale = kind(8192, dim, at, dim + at)
    cache = _cache(k8, v8, k_scale, v_scale)
    count = 50
    q = torch.zeros((count, 2, dim), dtype=dtype)
    q[..., 0] = 1
    out = torch.full_like(q, math.nan, device="cuda")
    kernels.attention_prefill_cache8(q.cuda(), cache, out, torch.arange(128, dtype=torch.int32)[None].cuda(), _ints([0, count]), _ints([8192 - count]), count, 1.0, impl, ranges)
    kernels.check_status()
    for i in range(count):
        seen = torch.arange(8192) <= 8192 - count + i
        want, bound = _expected((k8[:, 0] / 16).masked_fill(~seen, -math.inf), v8, v_scale, dtype)
        off = (out[i].double().cpu() - want).abs()
        assert bool((off <= bound).all()), f"query {i}: {float((off / bound).max())} of the bound"


# (key, element) of the values that are not numbers, in a prompt of 150 tokens behind 100: in the earlier tokens, at a page's first and last place, several in one element, the last
# token's; and what lies behind the last token
NANS = [[(40, 3)], [(100, 0), (100, 17)], [(127, 5), (128, 6)], [(249, 15)], [(130, 2), (200, 2), (201, 9)], [(250, 1), (255, 8)], []]


@pytest.mark.parametrize("impl,dtype,dim,heads", [("tc", BF16, 128, 4), ("tc", BF16, 64, 2), ("tc", BF16, 48, 6), ("mma", BF16, 128, 4), ("mma", BF16, 64, 6), ("mma", F32, 128, 2),
                                                  ("mma", F32, 256, 2), ("mma", BF16, 16, 16)])
@pytest.mark.parametrize("ranges", [1, 2, 3])
@pytest.mark.parametrize("sign", [0x7f, 0xff])
def test_a_value_that_is_no_number_reaches_its_element_of_the_queries_that_see_it(impl, dtype, dim, heads, ranges, sign):
    """One sequence for each of NANS, in one call; kv head 1 of two has the NaN."""
    from qwen_triton_b200.ops import kernels
    count, past, pages = 150, 100, 4
    gen = torch.Generator().manual_seed(dim)
    n = len(NANS)
    k8, v8 = ((torch.randn((n * pages, 2, PAGE, dim), generator=gen) * 90).clamp(-448, 448).to(E4M3).cuda() for _ in range(2))
    held = [t.view(torch.uint8).cpu().view(E4M3).double() * 2.0 ** -7 for t in (k8, v8)]
    for i, places in enumerate(NANS):
        for key, element in places:
            v8.view(torch.uint8)[i * pages + key // PAGE, 1, key % PAGE, element % dim] = sign
    cache = kernels.Cache8(k8, v8, *(torch.full((n * pages, 2), 2.0 ** -7, device="cuda") for _ in range(2)))
    table = torch.arange(n * pages, dtype=torch.int32).view(n, pages)
    q = torch.randn((n * count, heads, dim), generator=gen).to(dtype)
    out = torch.zeros_like(q, device="cuda")
    kernels.attention_prefill_cache8(q.cuda(), cache, out, table.cuda(), _ints([count * i for i in range(n + 1)]), _ints([past] * n), count, dim ** -0.5, impl, ranges)
    kernels.check_status()
    want, bound = plain.attention(q, *held, table, [count] * n, [past] * n, dim ** -0.5, 11 if dtype == BF16 else 20, impl == "tc")
    bound = bound + want.abs() * torch.finfo(dtype).eps / 2 * (1 + 2.0 ** -8) + 1e-30
    nan = torch.zeros_like(want, dtype=torch.bool).view(n, count, heads, dim)
    for i, places in enumerate(NANS):
        for key, element in places:
            nan[i, max(0, key - past):, heads // 2:, element % dim] = True
    nan = nan.view_as(want)
    out = out.double().cpu()
    assert torch.equal(out.isnan(), nan)
    off = (out - want).abs()[~nan]
    assert bool((off <= bound[~nan]).all()), f"{float((off / bound[~nan]).max())} of the bound"


@pytest.mark.parametrize("impl,dtype", [("tc", BF16), ("mma", BF16), ("mma", F32)])
def test_a_key_that_is_no_number_reaches_the_queries_that_see_it(impl, dtype):
    from qwen_triton_b200.ops import kernels
    count, past = 100, 30
    gen = torch.Generator().manual_seed(1)
    k8, v8 = ((torch.randn((3, 1, PAGE, 64), generator=gen) * 90).clamp(-448, 448).to(E4M3).cuda() for _ in range(2))
    cache = kernels.Cache8(k8, v8, *(torch.full((3, 1), 2.0 ** -7, device="cuda") for _ in range(2)))
    q = torch.randn((count, 2, 64), generator=gen).to(dtype).cuda()
    args = (_ints([[0, 1, 2]]), _ints([0, count]), _ints([past]), count, 0.125, impl)
    without, out = torch.empty_like(q), torch.empty_like(q)
    kernels.attention_prefill_cache8(q, cache, without, *args)
    k8.view(torch.uint8)[1, 0, 16, 5] = 0x7f               # key 80, token 50
    kernels.attention_prefill_cache8(q, cache, out, *args)
    assert torch.equal(out[:50], without[:50]) and bool(out[50:].isnan().all()) and bool(without.isfinite().all())


def test_sizes_beyond_what_tcgen05_takes_go_to_the_other_form(monkeypatch):
    """The limits made small: the default takes the form that has none, and a call that asks for tcgen05 is refused."""
    from qwen_triton_b200.ops import kernels
    gen = torch.Generator().manual_seed(2)
    k8, v8 = ((torch.randn((5, 2, PAGE, 64), generator=gen) * 90).clamp(-448, 448).to(E4M3).cuda() for _ in range(2))
    cache = kernels.Cache8(k8, v8, *(torch.full((5, 2), 2.0 ** -7, device="cuda") for _ in range(2)))
    q = torch.randn((300, 4, 64), generator=gen).to(BF16).cuda()
    args = (_ints([[0, 1, 2, 3, 4]]), _ints([0, 300]), _ints([20]), 300, 0.125)

    def call(impl):
        out = torch.empty_like(q)
        kernels.attention_prefill_cache8(q, cache, out, *args, impl)
        return out

    want, tc = call("mma"), call("tc")
    assert not torch.equal(want, tc)                       # what follows tells the forms apart
    monkeypatch.setattr(kernels, "prefill8_plan", lambda *a, on_tc, on_mma, **sizes: ("tc", 1) if on_tc else ("mma", 1))
    assert torch.equal(call(None), tc)
    for name, limit in (("_TC_PAGE_HEADS", 9), ("_TC_ROW_BLOCKS", 2)):
        with monkeypatch.context() as limits:
            limits.setattr(kernels, name, limit)
            assert torch.equal(call(None), want)
            with pytest.raises(kernels.KernelError, match="impl='tc'"):
                call("tc")


def test_operands_of_another_rank_are_refused():
    """As every other call that is not in order: with a KernelError, before anything is launched."""
    from qwen_triton_b200.ops import kernels
    cache = kernels.cache8(2, 1, 64, "cuda")
    q, out = (torch.zeros((2, 1, 64), device="cuda") for _ in range(2))
    qkv, table, start, past = kernels.GemmOut(torch.zeros((1, 2, 192), device="cuda")), _ints([[0], [1]]), _ints([0, 1, 2]), _ints([0, 0])
    plan = kernels.decode8_plan(2, num_heads=1, num_kv_heads=1, head_dim=64, dtype=F32, max_context=64)
    weight, rows, x, y = kernels.quantise_weight_fp8(torch.zeros((64, 32), device="cuda")), kernels.fp8_rows(2, 32, "cuda"), torch.zeros((2, 32), device="cuda"), torch.zeros((2, 64), device="cuda")
    calls = [(lambda *a: kernels.qkv_write_cache8(qkv, a[0], cache, *a[1:], 1, None, None, 1e-6, None), (q, start, past, table)),
             (lambda *a: kernels.attention_prefill_cache8(a[0], cache, *a[1:], 1, 0.1), (q, out, table, start, past)),
             (lambda *a: kernels.attention_decode_cache8(a[0], cache, *a[1:], 0.1, plan), (q, out, table, past)),
             (lambda *a: kernels.gemm_fp8(a[0], weight, a[1], rows), (x, y))]
    before = kernels.launch_count()
    for call, operands in calls:
        for i, operand in enumerate(operands):
            for other in (operand[None], operand.reshape(-1), operand.reshape(-1)[0]):
                if other.shape != operand.shape:
                    with pytest.raises(kernels.KernelError):
                        call(*operands[:i], other, *operands[i + 1:])
    assert kernels.launch_count() == before
    for call, operands in calls:
        call(*operands)
