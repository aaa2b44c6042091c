"""Products of an 8-bit weight: plans for the device, the cut of a last round, rows that are not finite."""
import math

import pytest
import torch

import plain_8bit as plain

pytestmark = pytest.mark.gpu
E4M3 = torch.float8_e4m3fn


def test_plans_are_for_the_device_s_multiprocessors(monkeypatch):
    """Not for a number that is written down: a device may have others, and the launch of a last round asks the device."""
    from qwen_triton_b200.ops import kernels
    asked = {}
    for name in ("fp8_plan", "fp8_last_round", "prefill8_plan"):
        def spy(*args, _name=name, _plan=getattr(kernels, name), **kwargs):
            asked[_name] = kwargs.get("sms", args[-1])
            return _plan(*args, **kwargs)
        monkeypatch.setattr(kernels, name, spy)
    device = torch.cuda.current_device()
    monkeypatch.setitem(kernels._SM_COUNTS, device, 132)
    weight = kernels.quantise_weight_fp8(torch.randn((512, 256), device="cuda"))
    x, rows = torch.randn((2000, 256), device="cuda"), kernels.fp8_rows(2000, 256, "cuda")
    out = torch.empty((2000, 512), device="cuda")
    kernels.gemm_fp8(x, weight, out, rows)
    kernels.gemm_fp8(x, weight, out, rows, (256, 1))
    q = torch.randn((4, 2, 64), dtype=torch.bfloat16, device="cuda")
    table, start, past = (torch.tensor(v, dtype=torch.int32, device="cuda") for v in ([[0]], [0, 4], [0]))
    kernels.attention_prefill_cache8(q, kernels.cache8(1, 1, 64, "cuda"), torch.empty_like(q), table, start, past, 4, 0.125)
    assert asked == {"fp8_plan": 132, "fp8_last_round": 132, "prefill8_plan": 132}


def _operands(m, n, k, seed):
    gen = torch.Generator().manual_seed(seed)
    x = torch.randn((m, k), generator=gen) * torch.where(torch.rand(k, generator=gen) < 0.02, 30.0, 1.0)
    values = (torch.randn((n, k), generator=gen) * 100).clamp(-448, 448).to(E4M3)
    return x, values, 1e-3 * torch.rand((-(-n // 128), -(-k // 128)), generator=gen) + 1e-5


@pytest.mark.parametrize("m,n,k", [(1275, 3833, 4080), (1512, 6335, 6800)])
@pytest.mark.parametrize("out_dtype", [torch.bfloat16, torch.float32])
def test_a_last_round_in_ranges_of_k(m, n, k, out_dtype):
    """Every tile from its own operands: a few tiles behind one or two full rounds, the last row and column of tiles not full."""
    from qwen_triton_b200.ops import kernels
    tiles = -(-m // 128) * -(-n // 256)
    ranges = kernels.fp8_last_round(m, n, k, kernels.sm_count())
    assert ranges > 1 and tiles > kernels.sm_count() and m % 128 and n % 256
    x, values, scales = _operands(m, n, k, m)
    x = x.to(torch.bfloat16)
    out = torch.full((m, n), math.nan, dtype=out_dtype, device="cuda")
    before = kernels.launch_count()
    kernels.gemm_fp8(x.cuda(), kernels.Fp8Weight(values.cuda(), scales.cuda()), out, kernels.fp8_rows(m, k, "cuda"), (256, 1))
    assert kernels.launch_count() - before == 3            # the rows to 8 bits, the full rounds, the last one
    kernels.check_status()
    x8, x_scale = plain.quantise_rows(x)
    want, bound = (t.cpu() for t in plain.product(x8.cuda(), x_scale.cuda(), values.double().cuda(), scales.cuda()))
    bound = bound + want.abs() * torch.finfo(out_dtype).eps / 2 * (1 + 2 ** -8)
    off = (out.double().cpu() - want).abs()
    assert bool((off <= bound).all()), f"{float((off / bound).max())} of the bound"


PLANS = [(0, 1), (16, 1), (16, 2), (16, 4), (32, 1), (64, 2), (256, 1), (256, 3), None]


@pytest.mark.parametrize("plan", PLANS)
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("given", [False, True])
def test_rows_that_are_not_finite(plan, dtype, given):
    """A row with an infinity or a NaN anywhere is NaN throughout, where the weight's block is zero too; the others are as without it.  By every form, rows brought to 8 bits on
    the way, before the product, and by the caller."""
    from qwen_triton_b200.ops import kernels
    m, n, k = 12, 300, 1040
    x, values, scales = _operands(m, n, k, 1)
    values.view(torch.uint8)[:128, :128] = 0
    x = x.to(dtype)
    clean = x.clone()
    for row, column, what in ((0, 5, math.inf), (3, 200, math.nan), (4, 100, -math.inf), (7, 1039, math.inf), (8, 1030, math.nan), (11, 0, -math.nan)):
        x[row, column] = what
    bad = ~x.isfinite().all(1)
    weight, rows = kernels.Fp8Weight(values.cuda(), scales.cuda()), kernels.fp8_rows(m, k, "cuda")
    outs = []
    for rows_in in (x.cuda(), clean.cuda()):
        outs.append(torch.full((m, n), 7.0, dtype=dtype, device="cuda"))
        if given:
            kernels.quantise_rows_fp8(rows_in, rows)
            kernels.gemm_fp8(rows, weight, outs[-1], plan=plan)
        else:
            kernels.gemm_fp8(rows_in, weight, outs[-1], rows, plan)
    kernels.check_status()
    assert bool(outs[0][bad].isnan().all())
    assert torch.equal(outs[0][~bad], outs[1][~bad]) and bool(outs[1].isfinite().all())


@pytest.mark.parametrize("m", [1, 5])
def test_a_few_rows_that_are_not_finite_brought_to_8_bits_on_the_way(m):
    """At most 16 groups a block: the summing warps bring the rows to 8 bits themselves."""
    from qwen_triton_b200.ops import kernels
    x, values, scales = _operands(m, 200, 384, 2)
    x[m - 1, 130] = math.inf
    out = torch.empty((m, 200), device="cuda")
    before = kernels.launch_count()
    kernels.gemm_fp8(x.cuda(), kernels.Fp8Weight(values.cuda(), scales.cuda()), out, kernels.fp8_rows(m, 384, "cuda"), (16, 1))
    assert kernels.launch_count() - before == 1
    assert bool(out[m - 1].isnan().all()) and bool(out[:m - 1].isfinite().all())
