"""The product of rows and a weight in 8 bits with a scale for each block of 128, and what brings both to 8 bits, against 64 bits."""
import math

import pytest
import torch

import plain_8bit as plain

pytestmark = pytest.mark.gpu
E4M3 = torch.float8_e4m3fn


def _rows(m, k, dtype, seed, outliers=True):
    gen = torch.Generator().manual_seed(seed)
    x = torch.randn((m, k), generator=gen)
    if outliers:
        x *= torch.where(torch.rand(k, generator=gen) < 0.02, 30.0, 1.0)
    return x.to(dtype)


def _weight(n, k, seed):
    """Values and scales as a checkpoint may hold them: scales that are no powers of two, a block of zeros, the largest numbers."""
    gen = torch.Generator().manual_seed(seed)
    values = (torch.randn((n, k), generator=gen) * 100).clamp(-448, 448).to(E4M3)
    scales = 1e-3 * torch.rand((-(-n // 128), -(-k // 128)), generator=gen) + 1e-5
    values.view(torch.uint8)[:min(n, 128), :min(k, 128)] = 0 if min(scales.shape) > 1 else values.view(torch.uint8)[:min(n, 128), :min(k, 128)]
    return values, scales


def _check_product(m, n, k, dtype, out_dtype=None, seed=0, plan=None):
    from qwen_triton_b200.ops import kernels
    x, (values, scales) = _rows(m, k, dtype, seed), _weight(n, k, seed + 1)
    out = torch.full((m, n), math.nan, dtype=out_dtype or dtype, device="cuda")
    weight = kernels.Fp8Weight(values.cuda(), scales.cuda())
    kernels.gemm_fp8(x.cuda(), weight, out, kernels.fp8_rows(m, k, "cuda"), plan)
    want, bound = plain.product(*plain.quantise_rows(x), values.double(), scales)
    bound = bound + want.abs() * torch.finfo(out.dtype).eps / 2 * (1 + 2 ** -8)
    off = (out.double().cpu() - want).abs()
    assert bool((off <= bound).all()), f"{float((off / bound.clamp(min=1e-300)).max())} of the bound"
    kernels.check_status()


@pytest.mark.parametrize("m", [1, 2, 3, 8, 9, 16, 17, 31, 33, 64, 65, 100, 128, 129, 200, 256, 257, 400])
@pytest.mark.parametrize("n,k", [(128, 128), (384, 512), (1000, 2832), (130, 272), (72, 1040)])
def test_product(m, n, k):
    _check_product(m, n, k, torch.bfloat16, seed=m)


@pytest.mark.parametrize("m,n,k", [(1, 1, 1), (5, 3, 7), (40, 129, 129), (3, 257, 100), (70, 65, 1000), (1, 127, 16), (300, 1, 48), (4, 24, 131)])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_product_of_odd_sizes(m, n, k, dtype):
    _check_product(m, n, k, dtype)


@pytest.mark.parametrize("m,n,k", [(1, 1024, 2048), (8, 512, 12288), (333, 640, 4096), (77, 1000, 2832), (600, 768, 1024)])
def test_product_in_float32(m, n, k):
    _check_product(m, n, k, torch.float32)
    _check_product(m, n, k, torch.bfloat16, torch.float32)
    _check_product(m, n, k, torch.float32, torch.bfloat16)


@pytest.mark.parametrize("m,n,k", [(1, 4096, 4096), (8, 6144, 4096), (700, 5120, 1024), (2048, 2560, 512)])
def test_product_of_many_tiles(m, n, k):
    _check_product(m, n, k, torch.bfloat16)


@pytest.mark.parametrize("form,splits", [(0, 1)] + [(form, splits) for form in (16, 32, 64, 256) for splits in (1, 2, 3, 5, 7, 8)])
@pytest.mark.parametrize("m,n,k", [(1, 130, 1040), (150, 300, 1040), (33, 256, 400), (129, 512, 112)])
def test_product_by_every_plan(form, splits, m, n, k):
    """Any plan gives the result, more ranges than K has blocks among them."""
    _check_product(m, n, k, torch.bfloat16, torch.float32, plan=(form, splits))
    _check_product(m, n, k, torch.bfloat16, plan=(form, splits))


def test_the_same_rows_give_the_same_bits():
    """Alone and twice, in 8 bits already or not: sums are in one order."""
    from qwen_triton_b200.ops import kernels
    for m, plan in ((48, None), (300, None), (4, (32, 2)), (20, (16, 3))):
        x, (values, scales) = _rows(m, 1152, torch.bfloat16, 3).cuda(), _weight(1024, 1152, 4)
        weight = kernels.Fp8Weight(values.cuda(), scales.cuda())
        rows = kernels.fp8_rows(m, 1152, "cuda")
        outs = [torch.empty((m, 1024), dtype=torch.bfloat16, device="cuda") for _ in range(3)]
        kernels.gemm_fp8(x, weight, outs[0], rows, plan)
        kernels.gemm_fp8(x, weight, outs[1], kernels.fp8_rows(m + 7, 1152, "cuda"), plan)
        kernels.quantise_rows_fp8(x, rows)
        kernels.gemm_fp8(rows, weight, outs[2], plan=plan)
        assert torch.equal(outs[0], outs[1]) and torch.equal(outs[0], outs[2])


@pytest.mark.parametrize("m,n,k", [(1, 256, 512), (3, 130, 2832), (5, 384, 2992), (16, 128, 1040)])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_rows_that_come_in_8_bits_give_the_same_bits(m, n, k, dtype):
    """Whether a product brings its rows to 8 bits on the way or finds them so, its sums are the same."""
    from qwen_triton_b200.ops import kernels
    x, (values, scales) = _rows(m, k, dtype, 3).cuda(), _weight(n, k, 4)
    weight = kernels.Fp8Weight(values.cuda(), scales.cuda())
    rows = kernels.fp8_rows(m, k, "cuda")
    kernels.quantise_rows_fp8(x, rows)
    for splits in (1, 2, 8):
        outs = [torch.empty((m, n), dtype=dtype, device="cuda") for _ in range(2)]
        kernels.gemm_fp8(x, weight, outs[0], kernels.fp8_rows(m, k, "cuda"), (16, splits))
        kernels.gemm_fp8(rows, weight, outs[1], plan=(16, splits))
        assert torch.equal(*outs)


def test_rows_and_sums_at_the_ends_of_the_range():
    """Rows of zeros, of the smallest and largest numbers, with an infinity or a NaN: such a row is NaN, the others are as without it."""
    from qwen_triton_b200.ops import kernels
    x = _rows(7, 512, torch.float32, 5)
    x[0] = 0
    x[1] *= 1e-38
    x[2] *= 1e30
    x[3, 200] = math.inf
    x[4, 300] = math.nan
    x[5, 100] = -math.inf
    values, scales = _weight(256, 512, 6)
    weight = kernels.Fp8Weight(values.cuda(), scales.cuda())
    out = torch.empty((7, 256), device="cuda")
    kernels.gemm_fp8(x.cuda(), weight, out, kernels.fp8_rows(7, 512, "cuda"))
    out = out.double().cpu()
    assert bool((out[0] == 0).all())
    for row in (3, 4):
        assert bool(out[row].isnan().all())
    assert bool(out[5].isnan().any())          # the weight's block of zeros times NaN is NaN as well
    want, bound = plain.product(*plain.quantise_rows(x), values.double(), scales)
    for row in (1, 2, 6):
        assert bool(((out[row] - want[row]).abs() <= bound[row] + want[row].abs() * 2.0 ** -24 + 2.0 ** -149).all())


@pytest.mark.parametrize("m,k", [(1, 128), (3, 1), (5, 130), (9, 1000), (130, 256), (2, 25600)])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_rows_in_8_bits(m, k, dtype):
    from qwen_triton_b200.ops import kernels
    x = _rows(m, k, dtype, k)
    rows = kernels.fp8_rows(m, k, "cuda")
    kernels.quantise_rows_fp8(x.cuda(), rows)
    values, scales = plain.quantise_rows(x)
    assert torch.equal(rows.scales.cpu(), scales)
    assert torch.equal(rows.values.double().cpu(), values)


@pytest.mark.parametrize("power", [-110, -90, -60, -59, -20, 0, 59, 60, 100, 119])
def test_quotients_next_to_borders(power):
    """Rows whose quotients lie on, just above and just below the borders of 8-bit numbers, at scales of every size: the division is float32's."""
    from qwen_triton_b200.ops import kernels
    g = torch.Generator().manual_seed(power)
    most = (torch.rand(600, generator=g) + 1) * 2.0 ** power                 # each group's largest number, and its scale
    scale = (most * plain.PER_TOP).clamp(min=2.0 ** -100)
    every = torch.arange(127, dtype=torch.uint8).view(torch.float8_e4m3fn).double()
    border = (every[1:] + every[:-1]) / 2
    pick = border[torch.randint(0, len(border), (600, 127), generator=g)]
    x = (pick * scale[:, None].double()).float()
    x = (x.view(torch.int32) + torch.randint(-2, 3, x.shape, generator=g, dtype=torch.int32)).clamp(min=0).view(torch.float32).clamp(max=most[:, None])
    x = torch.cat((most[:, None], torch.where(torch.rand(x.shape, generator=g) < 0.5, -x, x)), 1)
    x[:, 5], x[:, 6] = 0.0, -0.0
    rows = kernels.fp8_rows(600, 128, "cuda")
    kernels.quantise_rows_fp8(x.cuda(), rows)
    want = x / rows.scales.cpu().T
    assert torch.equal(rows.scales.cpu()[0], scale)
    assert torch.equal(rows.values.cpu().view(torch.uint8), want.clamp(-448, 448).to(torch.float8_e4m3fn).view(torch.uint8))


@pytest.mark.parametrize("m,k,group", [(1, 16, 0), (3, 160, 16), (9, 512, 16), (130, 528, 0), (17, 1536, 32), (8, 12288, 16)])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("activation,limit", [("silu", 0.0), ("capped", 1.5)])
def test_gated_rows_in_8_bits(m, k, group, dtype, activation, limit):
    """Bit by bit what the activation and the rows to 8 bits give one after the other; infinities and NaN among them."""
    from qwen_triton_b200.ops import kernels
    activation = kernels.CAPPED_GATE if activation == "capped" else activation
    x = _rows(m, 2 * k, dtype, k + m).cuda() * 3
    if m > 2:
        x[1, 5], x[2, k] = math.inf, math.nan
    gate_up = kernels.GemmOut(x[None])
    act, want, got = torch.empty((m, k), dtype=dtype, device="cuda"), kernels.fp8_rows(m, k, "cuda"), kernels.fp8_rows(m, k, "cuda")
    kernels.swiglu(gate_up, act, group, activation, limit)
    kernels.quantise_rows_fp8(act, want)
    kernels.swiglu_fp8(gate_up, got, group, activation, limit)
    assert torch.equal(got.scales.view(torch.int32), want.scales.view(torch.int32))
    assert torch.equal(got.values.view(torch.uint8), want.values.view(torch.uint8))


@pytest.mark.parametrize("m,k,planes", [(1, 16, 1), (3, 144, 0), (9, 1024, 3), (130, 4096, 1), (5, 8208, 2), (2, 16384, 1), (700, 512, 1), (600, 2064, 1)])
@pytest.mark.parametrize("dtype,delta_type", [(torch.bfloat16, torch.bfloat16), (torch.bfloat16, torch.float32), (torch.float32, torch.float32), (torch.float32, torch.bfloat16)])
def test_normed_rows_in_8_bits(m, k, planes, dtype, delta_type):
    """The stream with its addition, bit by bit; the rows within their roundings: e4m3's half step, the type's, and float32's in the row's factor (a sum of k squares in
    a tree: a few 2^-24, counted as 2^-20)."""
    from qwen_triton_b200.ops import kernels
    gen = torch.Generator().manual_seed(m + k)
    stream, weight = torch.randn((m, k), generator=gen) * torch.exp2(torch.randint(-3, 4, (m, 1), generator=gen).float()), 1 + 0.3 * torch.randn(k, generator=gen)
    delta = torch.randn((planes, m, k), generator=gen).to(delta_type) if planes else None
    rows, held = kernels.fp8_rows(m, k, "cuda"), stream.cuda()
    kernels.add_rmsnorm_fp8(held, kernels.GemmOut(delta.cuda()) if planes else None, weight.cuda(), 1e-6, rows, dtype)
    if planes:
        total = delta[0].float()
        for plane in delta[1:]:
            total = total + plane.float()
        stream = stream + total
    assert torch.equal(held.cpu(), stream)
    x = stream.double()
    want = x * torch.rsqrt((x * x).mean(1, keepdim=True) + 1e-6) * weight.double()
    groups = -(-k // 128)
    most = torch.stack([want[:, g * 128:(g + 1) * 128].abs().amax(1) for g in range(groups)])
    scales = rows.scales.cpu().double()
    half = torch.finfo(dtype).eps / 2
    assert bool(((scales - most / 448).abs() <= most / 448 * (half + 2.0 ** -20)).all())
    wide = scales.repeat_interleave(128, 0)[:k].T
    got = rows.values.cpu().view(torch.uint8).view(torch.float8_e4m3fn).double() * wide
    assert bool(((got - want).abs() <= want.abs() * (2.0 ** -4 + half + 2.0 ** -20) * (1 + 2.0 ** -8) + wide * 2.0 ** -10).all())


def test_normed_rows_refusals():
    from qwen_triton_b200.ops import kernels
    stream, weight = torch.zeros((4, 32), device="cuda"), torch.ones(32, device="cuda")
    rows = kernels.fp8_rows(4, 32, "cuda")
    kernels.add_rmsnorm_fp8(stream, None, weight, 1e-6, rows)
    assert int(rows.values.view(torch.uint8).max()) == 0
    for bad in ({"residual": stream[:3]}, {"residual": stream.bfloat16()}, {"weight": weight[:16].contiguous()}, {"delta": kernels.GemmOut(torch.zeros((1, 3, 32), device="cuda"))},
                {"dtype": torch.float16}, {"rows": kernels.fp8_rows(4, 48, "cuda")}):
        given = {"residual": stream, "delta": None, "weight": weight, "eps": 1e-6, "rows": rows, **bad}
        with pytest.raises(kernels.KernelError):
            kernels.add_rmsnorm_fp8(**given)
    with pytest.raises(kernels.KernelError, match="24 columns"):
        kernels.add_rmsnorm_fp8(torch.zeros((4, 24), device="cuda"), None, torch.ones(24, device="cuda"), 1e-6, kernels.fp8_rows(4, 24, "cuda"))


def test_gated_rows_refusals():
    from qwen_triton_b200.ops import kernels
    plane = kernels.GemmOut(torch.zeros((1, 4, 64), dtype=torch.bfloat16, device="cuda"))
    for rows, group, match in ((kernels.fp8_rows(4, 32, "cuda"), 24, "turns"), (kernels.fp8_rows(4, 48, "cuda"), 0, "for 4 x 48"), (kernels.fp8_rows(3, 32, "cuda"), 0, "for 3 x 32"),
                               (kernels.fp8_rows(4, 32, "cuda"), -16, "turns")):
        with pytest.raises(kernels.KernelError, match=match):
            kernels.swiglu_fp8(plane, rows, group)
    with pytest.raises(kernels.KernelError):
        kernels.swiglu_fp8(kernels.GemmOut(torch.zeros((1, 4, 36), dtype=torch.bfloat16, device="cuda")), kernels.fp8_rows(4, 18, "cuda"))
    with pytest.raises(kernels.KernelError):
        kernels.swiglu_fp8(kernels.GemmOut(torch.zeros((1, 4, 64), dtype=torch.float16, device="cuda")), kernels.fp8_rows(4, 32, "cuda"))


@pytest.mark.parametrize("n,k", [(128, 128), (1, 1), (130, 257), (384, 1024), (1000, 144), (33, 2832)])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_a_weight_in_8_bits(n, k, dtype):
    from qwen_triton_b200.ops import kernels
    w = _rows(n, k, dtype, n + k) * 0.02
    weight = kernels.quantise_weight_fp8(w.cuda())
    values, scales = plain.quantise_weight(w)
    assert torch.equal(weight.scales.cpu(), scales)
    assert torch.equal(weight.values.double().cpu(), values)


def test_captured_and_on_another_stream():
    from qwen_triton_b200.ops import kernels
    values, scales = _weight(512, 1024, 8)
    weight = kernels.Fp8Weight(values.cuda(), scales.cuda())
    x, out, rows = torch.zeros((24, 1024), dtype=torch.bfloat16, device="cuda"), torch.empty((24, 512), dtype=torch.bfloat16, device="cuda"), kernels.fp8_rows(24, 1024, "cuda")
    kernels.gemm_fp8(x, weight, out, rows)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        kernels.gemm_fp8(x, weight, out, rows)
    stream = torch.cuda.Stream()
    for seed in (1, 2):
        given = _rows(24, 1024, torch.bfloat16, seed)
        x.copy_(given)
        torch.cuda.synchronize()
        with torch.cuda.stream(stream):
            graph.replay()
        stream.synchronize()
        want, bound = plain.product(*plain.quantise_rows(given), values.double(), scales)
        assert bool(((out.double().cpu() - want).abs() <= bound + want.abs() * 2.0 ** -8).all())
        with torch.cuda.stream(stream):
            second = torch.empty_like(out)
            kernels.gemm_fp8(x, weight, second, kernels.fp8_rows(24, 1024, "cuda"))
        stream.synchronize()
        assert torch.equal(second, out)


@pytest.mark.parametrize("m,n,k", [(600_000, 128, 4096), (45_000, 51_200, 128)])
def test_offsets_beyond_32_bits(m, n, k):
    """Rows, and results, of more than 2^31 numbers: those of rows from all over are what these rows give by themselves."""
    from qwen_triton_b200.ops import kernels
    gen = torch.Generator(device="cuda").manual_seed(m)
    x = torch.randn((m, k), generator=gen, device="cuda", dtype=torch.bfloat16)
    weight = kernels.quantise_weight_fp8(torch.randn((n, k), generator=gen, device="cuda", dtype=torch.bfloat16))
    out, rows = torch.empty((m, n), dtype=torch.bfloat16, device="cuda"), kernels.fp8_rows(m, k, "cuda")
    kernels.gemm_fp8(x, weight, out, rows, (256, 1))
    pick = torch.cat((torch.arange(5), torch.tensor([m // 2, 2 ** 31 // max(n, k) - 1, 2 ** 31 // max(n, k) + 1]), torch.arange(m - 60, m))).cuda()
    few, want = kernels.fp8_rows(len(pick), k, "cuda"), torch.empty((len(pick), n), dtype=torch.bfloat16, device="cuda")
    kernels.gemm_fp8(x[pick], weight, want, few, (256, 1))
    assert torch.equal(out[pick], want) and bool(want.isfinite().all())
    assert torch.equal(rows.values.view(torch.uint8)[pick], few.values.view(torch.uint8)) and torch.equal(rows.scales[:, pick], few.scales)


@pytest.mark.parametrize("m,n,k,launches", [(1, 512, 1024, 1), (8, 512, 12288, 2), (333, 512, 1024, 2), (1512, 6335, 6800, 3), (1600, 4096, 4096, 2), (5, 64, 100, 2)])
def test_launches_are_counted(m, n, k, launches):
    """Rows brought to 8 bits on the way, by a launch of their own, and the last round of a large product."""
    from qwen_triton_b200.ops import kernels
    from test_gpu_launch_counts import kernels_of
    x, weight = torch.ones((m, k), dtype=torch.bfloat16, device="cuda"), kernels.quantise_weight_fp8(torch.ones((n, k), dtype=torch.bfloat16, device="cuda"))
    out, rows = torch.empty((m, n), dtype=torch.bfloat16, device="cuda"), kernels.fp8_rows(m, k, "cuda")
    assert kernels_of(lambda: kernels.gemm_fp8(x, weight, out, rows)) == (launches, launches)
    assert bool((out.float() - k).abs().max() <= k * 2.0 ** -8)            # 1 / s and s may each be rounded


def test_refusals():
    from qwen_triton_b200.ops import kernels
    Error = kernels.KernelError
    values, scales = (t.cuda() for t in _weight(256, 384, 9))
    weight = kernels.Fp8Weight(values, scales)
    with pytest.raises(Error, match="values"):
        kernels.Fp8Weight(values.float(), scales)
    with pytest.raises(Error, match="scales"):
        kernels.Fp8Weight(values, scales[:, :2])
    with pytest.raises(Error, match="contiguous"):
        kernels.Fp8Weight(values[:, :128], scales[:, :1].contiguous())
    x, out = torch.zeros((4, 384), device="cuda"), torch.empty((4, 256), device="cuda")
    rows = kernels.fp8_rows(4, 384, "cuda")
    with pytest.raises(Error, match="scratch"):
        kernels.gemm_fp8(x, weight, out)
    with pytest.raises(Error, match="scratch"):
        kernels.gemm_fp8(x, weight, out, kernels.fp8_rows(3, 384, "cuda"))
    with pytest.raises(Error, match="out"):
        kernels.gemm_fp8(x, weight, out[:, :100].contiguous(), rows)
    with pytest.raises(Error, match="neither"):
        kernels.gemm_fp8(x, weight, out.half(), rows)
    with pytest.raises(Error, match="neither"):
        kernels.gemm_fp8(x.half(), weight, out, rows)
    with pytest.raises(Error, match="rows"):
        kernels.gemm_fp8(kernels.fp8_rows(4, 128, "cuda"), weight, out)
    with pytest.raises(Error, match="CUDA"):
        kernels.gemm_fp8(x.cpu(), weight, out, rows)
    for plan in ((48, 1), (16, 0), (16, 9)):
        with pytest.raises(Error, match="plan"):
            kernels.gemm_fp8(x, weight, out, rows, plan)
    none = torch.empty((0, 256), device="cuda")
    kernels.gemm_fp8(x[:0], weight, none, rows)                # nothing to do
