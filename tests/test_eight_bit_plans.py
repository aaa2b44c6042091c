"""How products and attention in 8 bits are cut, and the plain statement of 8-bit numbers (no device needed)."""
import math

import pytest
import torch

import plain_8bit as plain
from qwen_triton_b200 import load_preset
from qwen_triton_b200.engine.engine import check_formats
from qwen_triton_b200.ops import kernels


def test_the_plain_rounding_is_the_nearest_number():
    every = torch.arange(256, dtype=torch.uint8).view(torch.float8_e4m3fn).double()
    every = every[every.isfinite()].unique()
    x = torch.cat((every, (every[1:] + every[:-1]) / 2, torch.randn(20000, generator=torch.Generator().manual_seed(1), dtype=torch.float64) * 100, torch.tensor([1e9, -1e9, 1e-9])))
    y = plain.as_e4m3(x)
    assert bool(torch.isin(y, every).all())
    nearest = (x.clamp(-448, 448)[:, None] - every[None]).abs().amin(1)
    assert torch.equal((x.clamp(-448, 448) - y).abs(), nearest)
    assert torch.equal(y, x.float().clamp(-448, 448).to(torch.float8_e4m3fn).double())          # ties to even
    assert bool(plain.as_e4m3(torch.tensor([math.inf, math.nan])).isnan().all())


@pytest.mark.parametrize("m", [1, 3, 16, 17, 33, 64, 65, 100, 333, 1000, 4096])
@pytest.mark.parametrize("n,k", [(1, 16), (128, 128), (1000, 2832), (1024, 2048), (4096, 12288), (51200, 5120), (77, 25600), (130, 100)])
def test_plans_of_products(m, n, k):
    form, splits = kernels.fp8_plan(m, n, k)
    assert form in kernels.FP8_FORMS and 1 <= splits <= 8 and (k % 16 == 0 or form == 0)
    groups = -(-k // 128)
    assert splits == 1 or groups // splits >= 1


@pytest.mark.parametrize("batch,heads,kv_heads,dim,dtype", [(1, 16, 8, 128, torch.bfloat16), (48, 32, 8, 128, torch.bfloat16), (256, 64, 8, 128, torch.bfloat16), (5, 16, 16, 96, torch.float32),
                                                            (32, 40, 2, 64, torch.bfloat16), (3, 4, 2, 256, torch.float32)])
@pytest.mark.parametrize("context", [0, 1, 64, 65, 700, 5000, 32000, 200000])
@pytest.mark.parametrize("most", [1, 2, 9, 64])
def test_plans_of_attention(batch, heads, kv_heads, dim, dtype, context, most):
    """Every page is in a range, scratch is asked for where ranges join through memory alone, and no more ranges than allowed."""
    plan = kernels.decode8_plan(batch, num_heads=heads, num_kv_heads=kv_heads, head_dim=dim, dtype=dtype, max_context=context, most_ranges=most)
    assert 1 <= plan.ranges <= most and plan.range_pages >= 1 and plan.ranges * plan.range_pages * 64 >= context
    assert plan.through_memory == (plan.ranges > 8 or (plan.ranges > 1 and not plan.clusters))
    assert (plan.acc_elements > 0) == plan.through_memory and plan.acc_elements in (0, batch * heads * plan.ranges * dim)


def test_refused_plans():
    for bad in ({"num_heads": 5}, {"num_kv_heads": 0}, {"max_context": -1}, {"dtype": torch.float16}, {"most_ranges": 0}):
        given = {"num_heads": 4, "num_kv_heads": 2, "head_dim": 64, "dtype": torch.bfloat16, "max_context": 100, **bad}
        with pytest.raises(kernels.KernelError):
            kernels.decode8_plan(2, **given)


def test_what_must_be_on_a_gpu_is_refused_on_the_host():
    values = torch.zeros((128, 128), dtype=torch.uint8).view(torch.float8_e4m3fn)
    for make in (lambda: kernels.Fp8Weight(values, torch.zeros((1, 1))), lambda: kernels.Fp8Rows(values, torch.zeros((1, 128))),
                 lambda: kernels.cache8(2, 1, 64, "cpu"), lambda: kernels.quantise_weight_fp8(torch.zeros((4, 4)))):
        with pytest.raises(kernels.KernelError, match="CUDA"):
            make()


def test_models_that_take_the_formats():
    assert check_formats(load_preset("tiny-a").model_spec(), None, None) == {}
    assert check_formats(load_preset("qwen3-8b").model_spec(), "fp8", "fp8") == {"weight_format": "fp8", "cache_format": "fp8"}
    with pytest.raises(ValueError, match="neither"):
        check_formats(load_preset("tiny-a").model_spec(), "fp4", None)
    for preset in ("lederax-tiny-a", "vunepel-tiny-a", "bisodra-tiny-a", "regupel-tiny-a", "misudra-tiny-a", "bizurax-tiny-a"):
        with pytest.raises(ValueError, match="another layer"):
            check_formats(load_preset(preset).model_spec(), None, "fp8")


@pytest.mark.parametrize("n_seqs,tokens,heads,kv_heads,dim,dtype", [(1, 1, 16, 8, 128, torch.bfloat16), (3, 900, 32, 8, 128, torch.bfloat16), (64, 4, 64, 8, 64, torch.bfloat16),
                                                                    (1, 4096, 16, 16, 96, torch.bfloat16), (2, 300, 4, 2, 256, torch.bfloat16), (5, 77, 6, 3, 48, torch.float32)])
@pytest.mark.parametrize("pages", [1, 2, 9, 300, 5000])
def test_plans_of_prompts(n_seqs, tokens, heads, kv_heads, dim, dtype, pages):
    """tcgen05 where it can, as many ranges as a cluster has blocks at most and never more than pages; what is not offered is not chosen."""
    shape = {"num_heads": heads, "num_kv_heads": kv_heads, "head_dim": dim, "dtype": dtype, "max_pages": pages}
    impl, ranges = kernels.prefill8_plan(n_seqs, tokens, **shape)
    assert impl in ("tc", "mma") and 1 <= ranges <= min(8, pages)
    assert impl == "mma" or (dtype == torch.bfloat16 and dim <= 128)
    assert kernels.prefill8_plan(n_seqs, tokens, **shape, on_tc=False)[0] == "mma"
    if dtype == torch.bfloat16 and dim <= 128:
        assert kernels.prefill8_plan(n_seqs, tokens, **shape, on_mma=False)[0] == "tc"


@pytest.mark.parametrize("m", [1, 128, 333, 1512, 1600, 4096, 100_000])
@pytest.mark.parametrize("n,k", [(6335, 6800), (4096, 4096), (51200, 5120), (256, 128), (2568, 1024)])
def test_last_rounds(m, n, k):
    """A last round is cut only where there is one behind a full one, into ranges that fit at once."""
    ranges, tiles = kernels.fp8_last_round(m, n, k), -(-n // 256) * -(-m // 128)
    assert 1 <= ranges <= 8
    if ranges > 1:
        assert tiles > 148 and 0 < tiles % 148 * ranges <= 130 and -(-k // 128) // ranges >= 8
