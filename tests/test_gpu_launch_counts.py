"""What the library says it launches is what a captured call holds."""
from __future__ import annotations

import dataclasses

import pytest
import torch

from qwen_triton_b200.ops import kernels

pytestmark = pytest.mark.gpu


def kernels_of(call) -> tuple[int, int]:
    """(kernel nodes of the call's graph, launches that were counted for it)."""
    from cuda.bindings import runtime
    call()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph(keep_graph=True)
    before = kernels.launch_count()
    with torch.cuda.graph(graph):
        call()
    counted = kernels.launch_count() - before
    error, nodes, *_, count = runtime.cudaGraphGetNodes(runtime.cudaGraph_t(int(graph.raw_cuda_graph())), 1 << 10)
    assert error == runtime.cudaError_t.cudaSuccess
    of_kernels = 0
    for node in nodes[:count]:
        error, kind = runtime.cudaGraphNodeGetType(node)
        assert error == runtime.cudaError_t.cudaSuccess
        of_kernels += kind == runtime.cudaGraphNodeType.cudaGraphNodeTypeKernel
    return of_kernels, counted


@pytest.mark.parametrize("rows, vocab, launches", [(1, 151936, 1), (8, 503, 1), (64, 151936, 1), (256, 151936, 2), (330, 20003, 2), (700, 8300, 2), (700, 8000, 1)])
def test_filtered_sampling(rows, vocab, launches):
    """More rows than get four blocks each, of a vocabulary that could have more, go through a second launch."""
    logits = torch.zeros((rows, vocab), device="cuda")
    f, k = torch.ones(rows, device="cuda"), torch.zeros(rows, dtype=torch.int32, device="cuda")
    half = 0.5 * f
    out = torch.empty_like(k)
    assert kernels_of(lambda: kernels.sample_filtered(logits, f, k, half, half, half, out)) == (launches, launches)


@pytest.mark.parametrize("dtype, dim, shared_ranges, launches", [(torch.bfloat16, 64, 0, 1), (torch.bfloat16, 64, 2, 2), (torch.float32, 64, 2, 2), (torch.bfloat16, 20, 1, 2)])
def test_attention_over_a_shared_prefix(dtype, dim, shared_ranges, launches):
    plan = kernels.shared_plan(2, num_heads=4, num_kv_heads=2, head_dim=dim, dtype=dtype, groups=1, most_members=2, most_shared=64, most_own=64)
    plan = dataclasses.replace(plan, shared_ranges=shared_ranges, own_ranges=1)
    q = torch.zeros((2, 4, dim), dtype=dtype, device="cuda")
    cache, out = torch.zeros((4, 2, 64, dim), dtype=dtype, device="cuda"), torch.empty_like(q)
    def ints(values):
        return torch.tensor(values, dtype=torch.int32, device="cuda")
    table, lengths, members, share = ints([[0, 1], [0, 2]]), ints([70, 80]), ints([0, 1]), ints([[0, 2, 64]])
    acc, ml = torch.empty(plan.acc_elements, device="cuda"), torch.empty(plan.ml_elements, device="cuda")
    assert kernels_of(lambda: kernels.attention_decode_shared(q, cache, cache, out, table, lengths, members, share, 2, 64, dim ** -0.5, plan, acc, ml)) == (launches, launches)
