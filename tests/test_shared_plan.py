"""The cut of attention over shared prefixes, and refusals that need no GPU."""
import pytest
import torch

from qwen_triton_b200.engine.step import shared_shape, tokens_not_again
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


def pays(groups, heads=32, kv_heads=8, dim=128, dtype=torch.bfloat16, page=64):
    return kernels.sharing_pays(tokens_not_again(groups), heads, kv_heads, dim, dtype, page)


def test_what_is_not_read_again_decides():
    """Of each group by itself, whatever else is in the batch: 50 MB of keys and values, 4,096 bytes a token at these sizes."""
    def rest(first, count):
        return list(range(first, first + count)), 0
    assert tokens_not_again([([0, 2, 3], 192), ([1], 0)]) == 384
    assert tokens_not_again([(list(range(8)), 2048), ([8, 9], 64), rest(10, 6)]) == 7 * 2048 + 64
    assert tokens_not_again([([0, 1], 640), ([], 0)]) == 640
    assert not pays([([0, 1], 64), rest(2, 254)])               # 256 KB
    assert not pays([([0, 1], 512), rest(2, 62)])
    assert not pays([([0, 1], 4096), rest(2, 60)])              # 16 MB
    assert not pays([([0, 1], 64)] * 32 + [rest(64, 192)])
    assert pays([([0, 1], 16384)]) and pays([([0, 1], 16384), rest(2, 254)])
    assert pays([(list(range(8)), 2048)]) and not pays([(list(range(8)), 1024)])
    assert pays([(list(range(4 * g, 4 * g + 4)), 1100) for g in range(4)])     # 13,200 tokens over four groups
    assert not pays([(list(range(17)), 4096)], heads=16, kv_heads=1)           # 32 MB; sixteen heads to a kv head want 122
    assert pays([(list(range(64)), 4096)], heads=16, kv_heads=1)


def test_the_kernel_that_would_run_decides():
    many = [(list(range(64)), 16384)]
    assert pays(many) and pays(many, heads=5, kv_heads=5, dim=64) and pays(many, heads=6, kv_heads=3, dim=40)
    for sizes in (dict(dim=256), dict(dim=160), dict(dim=20), dict(page=16), dict(dim=256, dtype=torch.float32)):
        assert not pays(many, **sizes)
    few = [([0, 1], 256)]                                       # 2 MB of float32
    assert pays(few, dtype=torch.float32) and pays(few, dtype=torch.float32, page=16) and not pays(few)
    assert not pays([([0, 1], 64)], dtype=torch.float32)


def test_shapes_leave_out_what_shares_nothing():
    """The most members are of a group that shares, so that sequences beside it do not widen the plan."""
    lengths = [5000] * 2 + [300] * 62
    assert shared_shape([([0, 1], 4096), (list(range(2, 64)), 0)], lengths) == (2, 2, 4096, 1024)
