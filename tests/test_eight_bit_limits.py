"""Which calls over an 8-bit cache tcgen05 can take (no device needed)."""
import math

import pytest
import torch

from qwen_triton_b200.ops import kernels

LARGEST = (2 ** 31 - 1) // 64


@pytest.mark.parametrize("dtype,dim,scale,page_heads,rows,takes", [
    (torch.bfloat16, 128, 0.1, 10, 1, True), (torch.bfloat16, 16, 0.1, LARGEST, 65535 * 256, True), (torch.bfloat16, 16, 0.1, LARGEST + 1, 1, False),
    (torch.bfloat16, 16, 0.1, 10, 65535 * 256 + 1, False), (torch.float32, 128, 0.1, 10, 1, False), (torch.bfloat16, 144, 0.1, 10, 1, False),
    (torch.bfloat16, 128, 0.0, 10, 1, False), (torch.bfloat16, 128, -0.1, 10, 1, False), (torch.bfloat16, 128, math.nan, 10, 1, False)])
def test_what_tcgen05_takes(dtype, dim, scale, page_heads, rows, takes):
    assert kernels.prefill8_tc_takes(dtype, dim, scale, page_heads, rows) is takes
