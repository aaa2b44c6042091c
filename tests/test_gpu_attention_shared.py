"""Attention over shared prefixes against a plain statement in 64 bits that knows nothing of what is shared."""
from __future__ import annotations

import dataclasses
import math

import pytest
import torch

from qwen_triton_b200.ops import kernels
from qwen_triton_b200.ops.kernels import KernelError

pytestmark = pytest.mark.gpu
PAGE = 64


class Case:
    """Sequences over a paged cache: ``groups`` lists (shared tokens, [tokens of each member's own]); own None: a sequence without keys.  Pages are in no
    order; every place of the cache that no sequence sees, and the page that unused table entries name, holds ``outside``."""

    def __init__(self, groups, heads, kv_heads, dim, dtype=torch.bfloat16, page=PAGE, seed=0, outside=float("nan"), spare_pages=2, at_end=False):
        gen = torch.Generator().manual_seed(seed)
        batch = sum(len(own) for _, own in groups)
        order = torch.randperm(batch, generator=gen).tolist()
        need = sum(shared // page + sum(-(-(shared + (o or 0)) // page) - shared // page + 1 for o in own) for shared, own in groups)
        total = need + 1 + spare_pages
        free = list(range(total))[-(need + 1):] if at_end else torch.randperm(total, generator=gen).tolist()
        barred = free.pop()
        self.lengths, tables, self.members, share = [0] * batch, [[]] * batch, [], []
        rows = []                                              # (page, slot) pairs that some sequence sees
        copies = []
        for shared, own in groups:
            share.append([len(self.members), len(own), shared])
            whole, part = [free.pop() for _ in range(shared // page)], None
            for tokens in own:
                i = order.pop()
                self.members.append(i)
                pages = list(whole)
                if shared % page:
                    pages.append(free.pop())
                    if part is None:
                        part = pages[-1]
                    else:
                        copies.append((part, pages[-1], shared % page))
                self.lengths[i] = 0 if tokens is None else shared + tokens
                while len(pages) * page < self.lengths[i]:
                    pages.append(free.pop())
                tables[i] = pages
                rows += [(pages[j // page], j % page) for j in range(max(self.lengths[i], shared))]
        width = max(1, max(len(t) for t in tables))
        self.table = torch.tensor([t + [barred] * (width - len(t)) for t in tables], dtype=torch.int32).cuda()
        self.k = torch.full((total, kv_heads, page, dim), outside, dtype=dtype, device="cuda")
        self.v = torch.full((total, kv_heads, page, dim), outside, dtype=dtype, device="cuda")
        if rows:
            at = torch.tensor(rows).cuda()
            for cache in (self.k, self.v):
                cache[at[:, 0], :, at[:, 1]] = torch.randn((len(rows), kv_heads, dim), generator=gen).to(dtype).cuda()
        for a, b, n in copies:
            self.k[b, :, :n], self.v[b, :, :n] = self.k[a, :, :n], self.v[a, :, :n]
        self.q = (1.5 * torch.randn((batch, heads, dim), generator=gen)).to(dtype).cuda()
        self.seq_len = torch.tensor(self.lengths, dtype=torch.int32).cuda()
        self.members_dev = torch.tensor(self.members, dtype=torch.int32).cuda()
        self.share = torch.tensor(share, dtype=torch.int32).cuda()
        self.heads, self.kv_heads, self.dim, self.dtype, self.page, self.batch = heads, kv_heads, dim, dtype, page, batch
        self.scale = dim ** -0.5
        own = [o or 0 for _, group in groups for o in group]
        self.plan = kernels.shared_plan(batch, num_heads=heads, num_kv_heads=kv_heads, head_dim=dim, dtype=dtype, groups=len(groups),
                                        most_members=max(len(o) for _, o in groups), most_shared=max(s for s, _ in groups), most_own=max(own), page_tokens=page)

    def run(self, plan=None, **changes):
        plan = plan or self.plan
        out = torch.full_like(self.q, 7.0)
        acc = torch.full((plan.acc_elements,), float("nan"), device="cuda")
        ml = torch.full((plan.ml_elements,), float("nan"), device="cuda")
        named = dict(q=self.q, k_cache=self.k, v_cache=self.v, out=out, block_table=self.table, seq_len=self.seq_len, members=self.members_dev,
                     share=self.share, num_kv_heads=self.kv_heads, page_tokens=self.page, scale=self.scale, plan=plan, part_acc=acc, part_ml=ml)
        named.update(changes)
        kernels.attention_decode_shared(**named)
        return named["out"]

    def check(self, out, only=None):
        """Every element within what the roundings allow: of a result (bfloat16: 2^-8 of it), of weights handed to the tensor cores (bfloat16:
        2^-8 of sum p |v|), of a score (d + 1 roundings of 2^-24 of sum |q k|), of sums over n keys, of exponentials (2^-21 each, numerator and sum)."""
        bits, unit = (2.0 ** -8, 2.0 ** -24) if self.dtype == torch.bfloat16 else (2.0 ** -24, 2.0 ** -24)
        for i in range(self.batch) if only is None else only:
            n = self.lengths[i]
            if n == 0:
                assert torch.equal(out[i], torch.zeros_like(out[i])), f"sequence {i} sees no key"
                continue
            j = torch.arange(n, device="cuda")
            page, slot = self.table[i].long()[j // self.page], j % self.page
            per = self.heads // self.kv_heads
            k = self.k[page, :, slot].double().repeat_interleave(per, dim=1)
            v = self.v[page, :, slot].double().repeat_interleave(per, dim=1)
            q = self.q[i].double()
            products = q[None] * k * self.scale
            weights = torch.softmax(products.sum(-1), dim=0)
            want = torch.einsum("nh,nhd->hd", weights, v)
            size = torch.einsum("nh,nhd->hd", weights, v.abs())
            score_error = (self.dim + 1) * unit * products.abs().sum(-1).amax(0)[:, None]
            bound = bits * want.abs() + (bits + 2 * score_error + (2 * n + 16) * unit + 2.0 ** -20) * size
            off = (out[i].double() - want).abs()
            assert bool((off <= bound).all()), f"sequence {i} of {n} keys: {float((off / bound).max()):.2f} of what is allowed"


SHAPES = [(4, 2, 64), (8, 1, 32), (5, 5, 64), (6, 3, 48), (32, 8, 128), (16, 16, 96), (10, 2, 80), (4, 4, 16), (3, 1, 112), (40, 2, 128), (2, 1, 8)]


@pytest.mark.parametrize("heads,kv_heads,dim", SHAPES)
def test_lengths_at_every_edge(heads, kv_heads, dim):
    groups = [(0, [1]), (1, [1, 2]), (63, [1, 1, 65]), (64, [64, 1]), (65, [3, 200]), (127, [1]), (128, [30, 33, 34]), (191, [0, 1]), (500, [13, 64, 129, 1])]
    case = Case(groups, heads, kv_heads, dim, seed=heads + dim)
    case.check(case.run())


@pytest.mark.parametrize("heads,kv_heads,dim", [(4, 2, 64), (6, 3, 48), (16, 8, 128), (3, 1, 200), (2, 2, 20), (8, 1, 256)])
def test_float32(heads, kv_heads, dim):
    case = Case([(0, [1, 40]), (63, [1, 2, 100]), (130, [7] * 9), (300, [0, 5])], heads, kv_heads, dim, torch.float32, seed=dim)
    case.check(case.run())


@pytest.mark.parametrize("heads,kv_heads,dim,page,dtype", [(4, 2, 160, 64, torch.bfloat16), (4, 2, 64, 16, torch.bfloat16), (4, 1, 256, 64, torch.bfloat16),
                                                           (2, 1, 20, 64, torch.bfloat16), (4, 2, 64, 48, torch.float32)])
def test_head_and_page_sizes_beyond_the_tensor_cores(heads, kv_heads, dim, page, dtype):
    case = Case([(70, [1, 20, 90]), (0, [5])], heads, kv_heads, dim, dtype, page=page, seed=3)
    case.check(case.run())


@pytest.mark.parametrize("members,heads,kv_heads,dim", [(33, 4, 1, 128), (40, 8, 2, 64), (129, 2, 2, 64), (17, 64, 8, 128), (64, 5, 1, 128)])
def test_more_rows_than_a_tile(members, heads, kv_heads, dim):
    case = Case([(333, [1 + 7 * i % 50 for i in range(members)])], heads, kv_heads, dim, seed=members)
    case.check(case.run())


def test_long_prefix_and_long_own_keys():
    case = Case([(9001, [700, 1, 65]), (5, [3000, 2500])], 8, 2, 128, seed=5)
    case.check(case.run())


def test_float32_from_odd_addresses():
    """Operands that start between the boundaries of wide loads."""
    case = Case([(70, [1, 20, 90]), (0, [5])], 4, 2, 64, torch.float32, seed=3)
    def moved(tensor):
        place = torch.empty(tensor.numel() + 1, dtype=tensor.dtype, device="cuda")[1:].view(tensor.shape)
        return place.copy_(tensor)
    out = moved(torch.zeros_like(case.q))
    case.run(q=moved(case.q), k_cache=moved(case.k), v_cache=moved(case.v), out=out)
    case.check(out)


def test_sequences_without_keys():
    case = Case([(100, [5, None, 7]), (0, [None]), (64, [None, None])], 8, 2, 64, seed=6)
    case.check(case.run())


@pytest.mark.parametrize("shared_ranges,own_ranges", [(1, 1), (1, 3), (7, 1), (5, 6), (24, 8)])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_every_cut_gives_the_result(shared_ranges, own_ranges, dtype):
    case = Case([(777, [1, 300, 64]), (0, [90]), (130, [2, 2])], 8, 2, 64, dtype, seed=7)
    case.check(case.run(dataclasses.replace(case.plan, shared_ranges=shared_ranges, own_ranges=own_ranges)))


@pytest.mark.parametrize("own_ranges,direct_warps", [(1, 1), (1, 4), (2, 3), (3, 6), (8, 2), (8, 4)])
@pytest.mark.parametrize("heads,kv_heads,dim", [(8, 2, 64), (6, 3, 48), (40, 2, 128), (5, 5, 80)])
def test_one_launch_over_all_keys_gives_the_result(own_ranges, direct_warps, heads, kv_heads, dim):
    case = Case([(777, [1, 300, 64]), (0, [90, None]), (130, [2, 2]), (9, [0, 1])], heads, kv_heads, dim, seed=7)
    case.check(case.run(dataclasses.replace(case.plan, shared_ranges=0, own_ranges=own_ranges, direct_warps=direct_warps)))


def test_scores_far_apart_and_one_key_far_above():
    """Running maxima that move by more than any rescaling step, upwards and downwards."""
    case = Case([(640, [100, 3])], 4, 2, 64, seed=8)
    ramp = torch.linspace(-6, 6, case.k.shape[0], device="cuda")[torch.randperm(case.k.shape[0], device="cuda")]
    seen = case.k.isnan()
    case.k = torch.where(seen, case.k, case.k * ramp[:, None, None, None].to(case.k.dtype))
    for i in range(3):
        case.k[case.table[0, 5], :, 10 + i] *= 20
    # members share pages, so what is equal stays equal; the copies of partly shared pages do not arise at 640 = 10 pages
    case.check(case.run())


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("direct", [False, True])
def test_shared_positions_are_read_through_the_first_members_list_only(dtype, direct):
    """The other members' lists name pages of anything below the shared length, and what their own page holds below it counts for nothing."""
    case = Case([(200, [40, 3, 100]), (64, [1, 70])], 8, 2, 64, dtype, seed=12)
    want = case.run().clone()
    case.check(want)
    barred = case.k.shape[0] - 1
    plan = dataclasses.replace(case.plan, shared_ranges=0, own_ranges=2, direct_warps=3) if direct and dtype == torch.bfloat16 else case.plan
    truth = case.table.clone(), case.k.clone(), case.v.clone()
    for first, count, shared in case.share.tolist():
        for i in case.members[first + 1:first + count]:
            if shared % PAGE:
                page = int(case.table[i, shared // PAGE])
                case.k[page, :, :shared % PAGE] = float("nan")
                case.v[page, :, :shared % PAGE] = float("nan")
            case.table[i, :shared // PAGE] = barred
    out = case.run(plan)
    case.table, case.k, case.v = truth
    case.check(out)


def test_the_same_call_gives_the_same_bits_and_follows_its_stream():
    case = Case([(1000, [33] * 24), (0, [100, 2])], 32, 8, 128, seed=9)
    first = case.run().clone()
    assert torch.equal(first, case.run())
    stream = torch.cuda.Stream()
    late = torch.zeros_like(case.q)
    with torch.cuda.stream(stream):
        torch.cuda._sleep(2_000_000)
        late.copy_(case.q)                                    # the call must wait for its own stream's work
        out = case.run(q=late)
    stream.synchronize()
    assert torch.equal(first, out)


def test_a_captured_call_follows_new_lengths():
    """What a plan was made for is a limit; the lengths are read when the call runs."""
    case = Case([(700, [64, 200, 1])], 8, 2, 128, seed=10)
    out = torch.zeros_like(case.q)
    acc, ml = torch.empty(case.plan.acc_elements, device="cuda"), torch.empty(case.plan.ml_elements, device="cuda")
    case.run(out=out, part_acc=acc, part_ml=ml)
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        case.run(out=out, part_acc=acc, part_ml=ml)
    graph.replay()
    case.check(out)
    case.share.copy_(torch.tensor([[0, 3, 600]], dtype=torch.int32))          # fewer shared tokens, shorter sequences
    case.lengths = [min(n, 650 + 3 * i) for i, n in enumerate(case.lengths)]
    case.seq_len.copy_(torch.tensor(case.lengths, dtype=torch.int32))
    graph.replay()
    case.check(out)


def test_offsets_beyond_32_bits():
    """Pages at the end of a cache of more than 2^31 elements."""
    pages = 2 ** 31 // (8 * PAGE * 128) + 40
    free, _ = torch.cuda.mem_get_info()
    if free < 3 * pages * 8 * PAGE * 128 * 2:
        pytest.skip("not enough free memory")
    case = Case([(130, [1, 70])], 16, 8, 128, seed=11, outside=0.0, spare_pages=pages - 12, at_end=True)
    assert int(case.table.max()) * 8 * PAGE * 128 > 2 ** 31
    case.check(case.run())


def test_no_sequences():
    case = Case([(3, [1])], 4, 2, 64)
    plan = kernels.shared_plan(0, num_heads=4, num_kv_heads=2, head_dim=64, dtype=torch.bfloat16, groups=1, most_members=0, most_shared=0, most_own=0)
    case.run(plan, q=case.q[:0], out=case.q[:0].clone(), block_table=case.table[:0], seq_len=case.seq_len[:0], members=case.members_dev[:0])


def test_refusals():
    case = Case([(70, [1, 5])], 4, 2, 64)
    for changes, words in (
            (dict(q=case.q.float()), "bfloat16|float32"),
            (dict(q=case.q.transpose(0, 1)), "contiguous"),
            (dict(q=case.q.cpu()), "CUDA"),
            (dict(out=case.q[:1].clone()), "shape"),
            (dict(v_cache=case.v[..., :32].contiguous()), "values|value|shape"),
            (dict(block_table=case.table[:1]), "block_table"),
            (dict(block_table=case.table.long()), "int32"),
            (dict(seq_len=case.seq_len.long()), "int32"),
            (dict(members=case.members_dev[:1]), "shape"),
            (dict(share=case.share[:, :2].contiguous()), "shape"),
            (dict(num_kv_heads=4), "cache shape"),
            (dict(page_tokens=32), "cache shape"),
            (dict(plan=dataclasses.replace(case.plan, page_tokens=16)), "plan"),
            (dict(part_acc=torch.empty(3, device="cuda")), "scratch"),
            (dict(part_ml=torch.empty(3, device="cuda")), "scratch"),
            (dict(plan=dataclasses.replace(case.plan, num_heads=8)), "plan")):
        with pytest.raises(KernelError, match=words):
            case.run(**changes)
    for changes in (dict(shared_ranges=-1), dict(own_ranges=0), dict(shared_ranges=1 << 20), dict(shared_ranges=0, own_ranges=9), dict(shared_ranges=0, direct_warps=7),
                    dict(shared_ranges=0, direct_warps=0)):
        with pytest.raises(KernelError):
            plan = dataclasses.replace(case.plan, **changes)
            case.run(plan, part_acc=torch.empty(max(plan.acc_elements, 1), device="cuda"), part_ml=torch.empty(max(plan.ml_elements, 1), device="cuda"))
    with pytest.raises(KernelError, match="aligned"):
        case.run(part_acc=torch.empty(case.plan.acc_elements + 1, device="cuda")[1:])
    wide = Case([(70, [1, 5])], 40, 2, 128)                   # more shared memory than a block has
    with pytest.raises(KernelError, match="shared memory"):
        wide.run(dataclasses.replace(wide.plan, shared_ranges=0, own_ranges=8, direct_warps=6))
    wide.check(wide.run())                                    # and nothing of that stays behind


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_a_refused_call_launches_nothing(dtype):
    """More sequences than the second launch takes: the first has not run either."""
    n = 65536
    plan = kernels.shared_plan(n, num_heads=1, num_kv_heads=1, head_dim=8, dtype=dtype, groups=1, most_members=2, most_shared=64, most_own=1)
    plan = dataclasses.replace(plan, shared_ranges=1, own_ranges=1)
    q, cache = torch.zeros((n, 1, 8), dtype=dtype, device="cuda"), torch.zeros((2, 1, 64, 8), dtype=dtype, device="cuda")
    table, lengths = torch.zeros((n, 2), dtype=torch.int32, device="cuda"), torch.full((n,), 65, dtype=torch.int32, device="cuda")
    members, share = torch.arange(n, dtype=torch.int32, device="cuda"), torch.tensor([[0, 2, 64]], dtype=torch.int32, device="cuda")
    acc, ml, out = torch.full((plan.acc_elements,), 7.0, device="cuda"), torch.full((plan.ml_elements,), 7.0, device="cuda"), torch.full_like(q, 7.0)
    with pytest.raises(KernelError, match="too many"):
        kernels.attention_decode_shared(q, cache, cache, out, table, lengths, members, share, 1, 64, 0.5, plan, acc, ml)
    torch.cuda.synchronize()
    assert all(bool((x == 7).all()) for x in (acc, ml, out))
