"""Calls of the operators for drafted tokens and selected pages that share what they are given: one tensor as both caches,
one workspace for several captured executors, one kv head for hundreds of query heads."""
from __future__ import annotations

import pytest
import torch

import test_gpu_draft_attention as draft
import test_gpu_sparse_attention as sparse

pytestmark = pytest.mark.gpu
F16, BF16 = torch.float16, torch.bfloat16
ops = draft.ops


@pytest.mark.parametrize("S", [3, 25, 90])
def test_one_tensor_as_both_caches(ops, device, S):
    a = draft.make(device, 2, S, 8, 2, 64, 16, 400, BF16)
    want = ops.draft_attention(*{**a, "v_cache": a["k_cache"].clone()}.values())
    got = ops.draft_attention(*{**a, "v_cache": a["k_cache"]}.values())
    assert all(torch.equal(x, y) for x, y in zip(got, want))
    b = sparse.make(device, 2, 8, 2, 64, 16, 400, BF16)
    want = ops.sparse_attention(*{**b, "v_cache": b["k_cache"].clone()}.values(), 7)
    got = ops.sparse_attention(*{**b, "v_cache": b["k_cache"]}.values(), 7)
    assert all(torch.equal(x, y) for x, y in zip(got, want))


def test_one_workspace_for_several_graphs(pkg, ops, device):
    """Launches that follow each other may share a workspace: what one leaves there means nothing to the next."""
    a = draft.make(device, 2, 20, 8, 2, 128, 16, 3000, BF16)
    b = sparse.make(device, 3, 16, 2, 128, 16, 4000, BF16)
    paged = b["q"], b["k_cache"], b["v_cache"], b["table"], b["lengths"]
    sizes = [pkg.DraftAttentionOp(**a).workspace_size, pkg.SparseAttentionOp(*b.values(), 60).workspace_size,
             pkg.SparseAttentionOp(*b.values(), 9).workspace_size, pkg.PagedAttentionOp(*paged).workspace_size]
    ws = torch.randint(0, 256, (max(sizes),), dtype=torch.uint8, device=device)
    made = [pkg.DraftAttentionOp(**a, workspace=ws), pkg.SparseAttentionOp(*b.values(), 60, workspace=ws),
            pkg.SparseAttentionOp(*b.values(), 9, workspace=ws), pkg.PagedAttentionOp(*paged, workspace=ws)]
    want = [ops.draft_attention(*a.values()), ops.sparse_attention(*b.values(), 60), ops.sparse_attention(*b.values(), 9),
            ops.paged_attention(*paged)]
    graphs = []
    for op in made:
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[-1]):
            op.launch()
    for order in ((0, 1, 2, 3), (3, 2, 1, 0), (1, 1, 3, 3), (2, 0, 2, 0), (0, 3, 1, 2)):
        for op in made:
            op.out.fill_(7)
        for x in order:
            graphs[x].replay()
        torch.cuda.synchronize()
        for x in order:
            assert torch.equal(made[x].out, want[x][0]) and torch.equal(made[x].lse, want[x][1]), (order, x)


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("heads", [300, 1000])
def test_hundreds_of_query_heads_to_one(ops, device, dtype, heads):
    draft.check(ops, draft.make(device, 2, 3, heads, 1, 64, 16, 150, dtype))
    sparse.check(ops, sparse.make(device, 2, heads, 1, 64, 16, 300, dtype), 6)
