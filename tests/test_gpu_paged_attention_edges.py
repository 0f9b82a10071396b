"""paged_attention where it could go wrong unseen: long-lived graphs, scores and values at the ends of their types."""
from __future__ import annotations

import math

import pytest
import torch

import serve_ref as ref

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


def _near(out, lse, want):
    w_out, w_lse, b_out, b_lse = want
    off, l_off = (out.cpu().double() - w_out).abs(), (lse.cpu().double() - w_lse).abs()
    assert (off <= b_out).all(), f"out: {(off / b_out).max():.3g} of its bound"
    assert (l_off <= b_lse).all(), f"lse: {(l_off / b_lse).max():.3g} of its bound"


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("gap", [8, 12, 14, 15, 16, 17, 18, 24])
@pytest.mark.parametrize("B,heads,kv_heads,d,n", [
    (600, 2, 1, 64, 512),  # each wave alone
    (1, 2, 1, 64, 8192), (1, 4, 4, 96, 700), (2, 32, 1, 128, 8192), (1, 16, 1, 256, 4000)])
def test_one_key_far_above_the_others(ops, device, B, heads, kv_heads, d, n, gap, dtype):
    """A key whose score is `gap` above the others' and whose value is 0: the output is the sum of many small weights.
    The bound is serve_ref's: a weight's error is 2^-16 of it where it is at least 2^-24 of the largest; below that
    8192 keys' errors of 2^-40 and values up to 4 are less than half of the type's smallest spacing."""
    g = torch.Generator().manual_seed(gap * n + d)
    page = 16
    pages = -(-n // page)
    q = 0.02 * torch.randn(1, heads, d, generator=g)
    k, v = torch.randn(pages, page, kv_heads, d, generator=g), torch.randn(pages, page, kv_heads, d, generator=g)
    v.clamp_(-4, 4)
    q[..., 0] = 1
    k[..., 0] = 0
    at = n // 3
    k[at // page, at % page] = 0
    k[at // page, at % page, :, 0] = gap
    v[at // page, at % page] = 0
    q, k, v = (x.to(dtype).to(device) for x in (q, k, v))
    table = torch.arange(pages, dtype=torch.int32, device=device).view(1, -1)
    lengths = torch.tensor([n], dtype=torch.int32, device=device)
    out, lse = ops.paged_attention(q.expand(B, -1, -1).contiguous(), k, v, table.expand(B, -1).contiguous(),
                                   lengths.expand(B).contiguous(), 1.0)
    _near(out[-1:], lse[-1:], ref.attention(q, k, v, table, lengths, 1.0))


@pytest.mark.parametrize("scale", [1.0, 0.0, -0.125])
@pytest.mark.parametrize("B", [1, 300])
def test_extreme_scores_in_fp16(ops, device, B, scale):
    """Scores hundreds apart, equal ones, and the order turned round."""
    g = torch.Generator().manual_seed(B)
    q = 30 * torch.randn(1, 4, 64, generator=g)
    k, v = torch.randn(33, 16, 2, 64, generator=g), 100 * torch.randn(33, 16, 2, 64, generator=g)
    q, k, v = (x.half().to(device) for x in (q, k, v))
    table = torch.arange(32, dtype=torch.int32, device=device).view(1, -1)
    lengths = torch.tensor([509], dtype=torch.int32, device=device)
    out, lse = ops.paged_attention(q.expand(B, -1, -1).contiguous(), k, v, table.expand(B, -1).contiguous(),
                                   lengths.expand(B).contiguous(), scale)
    _near(out[-1:], lse[-1:], ref.attention(q, k, v, table, lengths, scale))


def test_the_longest_rows_there_may_be(ops, device):
    """2^31 - 2 keys in two pages whose slots are one and the same memory.  The window's keys are equal but for the
    last case's 50 from the page before (weights of e^-9 beside 2^30 of 1); lse is off by at most eight roundings."""
    page = 2 ** 30 - 1
    rows = torch.zeros(2, 2, 1, 1, 32)
    rows[0, 1, ..., 0], rows[0, 0, ..., 0] = 16, -2  # scores 8 and -1
    rows[1] = torch.arange(64).view(2, 1, 1, 32)
    k, v = (r.to(torch.bfloat16).to(device).expand(2, page, 1, 32) for r in rows)
    q = torch.zeros(1, 1, 32, dtype=torch.bfloat16, device=device)
    q[..., 0] = 1
    table = torch.tensor([[0, 1]], dtype=torch.int32, device=device)
    for length, window, keys in ((2 * page, 100, 100), (2 * page, 1, 1), (2 ** 31 - 1, 1000, 1000),
                                 (2 * page, page + 50, page)):
        lengths = torch.tensor([length], dtype=torch.int32, device=device)
        out, lse = ops.paged_attention(q, k, v, table, lengths, 0.5, window)
        assert torch.equal(out[0, 0], v[1, 0, 0])
        want = 8 + math.log(keys)
        assert abs(float(lse) - want) <= 8 * 2.0 ** -24 * (1 + want)
    out, lse = ops.paged_attention(q, k, v, torch.full_like(table, -1), lengths, 0.5)  # holes only
    assert (out == 0).all() and torch.isneginf(lse).all()
