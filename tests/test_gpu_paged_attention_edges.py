"""paged_attention where it could go wrong unseen: long-lived graphs, scores and values at the ends of their types."""
from __future__ import annotations

import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ops(pkg, device):
    pkg.torch_ops()
    return torch.ops.mhcpre


@pytest.mark.parametrize("heads,kv_heads,first,then", [(8, 2, 3000, 3000), (8, 2, 3000, 5000), (8, 2, 5000, 3000),
                                                       (1, 1, 66000, 66000), (1, 1, 66000, 40000)])
def test_counts_of_old_replays_are_gone(pkg, ops, device, heads, kv_heads, first, then):
    """A captured launch on a workspace of its own: a replay that joins parts, 2047 that have none, and one that joins
    again, under the number that the first one had (a replay's number has 11 bits).  Rows in spans, too."""
    g = torch.Generator(device=device).manual_seed(first)
    page, d = 64, 64
    pages = -(-max(first, then) // page)
    q = torch.randn(1, heads, d, generator=g, device=device).to(torch.bfloat16)
    k, v = (torch.randn(pages, page, kv_heads, d, generator=g, device=device).to(torch.bfloat16) for _ in range(2))
    table = torch.randperm(pages, generator=g, device=device).int().view(1, pages)
    lengths = torch.tensor([first], dtype=torch.int32, device=device)
    op = pkg.PagedAttentionOp(q, k, v, table, lengths)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        op.launch()
    for n, replays in ((first, 1), (0, 2047), (then, 1), (0, 2047), (first, 1)):
        lengths.fill_(n)
        for _ in range(replays - 1):
            graph.replay()
        op.out.fill_(7)
        op.lse.fill_(7)
        graph.replay()
        torch.cuda.synchronize()
        want = ops.paged_attention(q, k, v, table, lengths)
        assert torch.equal(op.out, want[0]) and torch.equal(op.lse, want[1]), n
