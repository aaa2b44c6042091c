"""Which models take an 8-bit cache, and which calls over one tcgen05 can take (no device needed)."""
import dataclasses
import math

import pytest
import torch

from qwen_triton_b200 import load_preset
from qwen_triton_b200.config.spec import LayerCall
from qwen_triton_b200.engine.engine import check_formats
from qwen_triton_b200.ops import kernels

LARGEST = (2 ** 31 - 1) // 64


@pytest.mark.parametrize("dtype,dim,scale,page_heads,rows,takes", [
    (torch.bfloat16, 128, 0.1, 10, 1, True), (torch.bfloat16, 16, 0.1, LARGEST, 65535 * 256, True), (torch.bfloat16, 16, 0.1, LARGEST + 1, 1, False),
    (torch.bfloat16, 16, 0.1, 10, 65535 * 256 + 1, False), (torch.float32, 128, 0.1, 10, 1, False), (torch.bfloat16, 144, 0.1, 10, 1, False),
    (torch.bfloat16, 128, 0.0, 10, 1, False), (torch.bfloat16, 128, -0.1, 10, 1, False), (torch.bfloat16, 128, math.nan, 10, 1, False)])
def test_what_tcgen05_takes(dtype, dim, scale, page_heads, rows, takes):
    assert kernels.prefill8_tc_takes(dtype, dim, scale, page_heads, rows) is takes


def test_calls_that_read_another_call_s_cache_are_refused():
    """Such a call writes nothing; the write into an 8-bit cache would put its own keys and values over the other call's."""
    spec = load_preset("tiny-a").model_spec()
    reader = dataclasses.replace(spec, schedule=[LayerCall(0), LayerCall(1, cache_of=0)])
    reader.validate()
    with pytest.raises(ValueError, match="reads another's"):
        check_formats(reader, None, "fp8")
    assert check_formats(reader, "fp8", None) == {"weight_format": "fp8"}
    twice = dataclasses.replace(spec, schedule=[LayerCall(0), LayerCall(1), LayerCall(0)])                # entries of their own
    assert check_formats(twice, None, "fp8") == {"cache_format": "fp8"}
