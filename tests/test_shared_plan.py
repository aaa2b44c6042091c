"""The cut of attention over shared prefixes, and refusals that need no GPU."""
import pytest
import torch

from qwen_triton_b200.ops import kernels
from qwen_triton_b200.ops.kernels import KernelError


def plan(n_seqs=8, groups=1, most_members=8, most_shared=2048, most_own=100, heads=32, kv_heads=8, dim=128, dtype=torch.bfloat16, sms=148):
    return kernels.shared_plan(n_seqs, num_heads=heads, num_kv_heads=kv_heads, head_dim=dim, dtype=dtype, groups=groups, most_members=most_members,
                               most_shared=most_shared, most_own=most_own, sms=sms)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_every_size_has_a_cut_whose_scratch_is_bounded(dtype):
    for n_seqs in (1, 2, 7, 64, 256):
        for shared in (0, 1, 63, 64, 1000, 40960):
            for own in (0, 1, 500, 40960):
                for heads, kv_heads, dim in ((16, 8, 128), (64, 8, 128), (5, 5, 64), (8, 1, 32)):
                    p = plan(n_seqs, min(n_seqs, 3), n_seqs, shared, own, heads, kv_heads, dim, dtype)
                    assert p.shared_ranges >= 0 and p.own_ranges >= 1 and (p.shared_ranges or dtype == torch.bfloat16)
                    assert p.acc_elements == n_seqs * heads * p.ranges * dim and p.ml_elements == 2 * n_seqs * heads * p.ranges
                    assert p.ranges <= 64


def test_refusals():
    for wrong in (dict(groups=0), dict(most_members=9), dict(most_shared=-1), dict(most_own=-1), dict(heads=30), dict(dim=0), dict(dtype=torch.float16)):
        with pytest.raises(KernelError):
            plan(**wrong)


def test_there_is_no_host_path():
    p = plan(1, 1, 1, 64, 1, 4, 2, 64)
    q, cache = torch.zeros((1, 4, 64), dtype=torch.bfloat16), torch.zeros((2, 2, 64, 64), dtype=torch.bfloat16)
    one = torch.zeros(1, dtype=torch.int32)
    with pytest.raises(KernelError, match="host"):
        kernels.attention_decode_shared(q, cache, cache, q, one[None], one, one, one.repeat(3)[None], 2, 64, 0.125, p, torch.zeros(9999), torch.zeros(9999))
    with pytest.raises(KernelError, match="host"):
        f = torch.zeros(1)
        kernels.sample_filtered(torch.zeros((1, 5)), f, one, f, f, f, one)
