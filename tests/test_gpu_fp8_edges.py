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
