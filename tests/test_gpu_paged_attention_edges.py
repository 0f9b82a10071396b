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


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("B,heads,kv_heads,d,n", [(1, 2, 1, 64, 1), (600, 2, 1, 64, 100), (1, 4, 2, 96, 3000),
                                                  (2, 32, 1, 128, 300), (1, 5, 1, 256, 700)])
def test_infinite_and_nan_values(ops, device, B, heads, kv_heads, d, n, dtype):
    """A value that a row sees is infinite or NaN: so is the output's column, and no other one."""
    g = torch.Generator().manual_seed(n + d)
    page = 16
    pages = -(-n // page) + 1
    q = torch.randn(1, heads, d, generator=g)
    k, v = torch.randn(pages, page, kv_heads, d, generator=g), torch.randn(pages, page, kv_heads, d, generator=g)
    finite = v.clone()

    def put(t, column, value):
        v[t // page, t % page, :, column], finite[t // page, t % page, :, column] = value, 0

    put(n // 3, 3, math.inf)
    put(n // 2, 17, -math.inf)
    put(n - 1, d - 1, math.nan)
    put(0, 9, math.inf)
    put(n - 1, 9, math.inf)
    put(0, 12, -math.inf if n == 1 else math.inf)
    if n > 1:
        put(n - 1, 12, -math.inf)
    v[pages - 1], finite[pages - 1] = math.nan, 0  # nobody's
    q, k, v, finite = (x.to(dtype).to(device) for x in (q, k, v, finite))
    table = torch.arange(pages - 1, dtype=torch.int32, device=device).view(1, -1)
    lengths = torch.tensor([n], dtype=torch.int32, device=device)
    out, lse = ops.paged_attention(q.expand(B, -1, -1).contiguous(), k, v, table.expand(B, -1).contiguous(),
                                   lengths.expand(B).contiguous())
    last = out[-1].cpu().double()
    assert (last[:, 3] == math.inf).all() and (last[:, 17] == -math.inf).all() and torch.isnan(last[:, d - 1]).all()
    assert (last[:, 9] == math.inf).all()
    assert (last[:, 12] == -math.inf).all() if n == 1 else torch.isnan(last[:, 12]).all()
    want = ref.attention(q, k, finite, table, lengths, d ** -0.5)
    rest = [c for c in range(d) if c not in (3, 9, 12, 17, d - 1)]
    _near(out[-1:, :, rest], lse[-1:], (want[0][..., rest], want[1], want[2][..., rest], want[3]))


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_infinite_value_of_a_small_weight(ops, device, dtype):
    """A weight of e^-40 beside the largest is not 0 in 32 bits: its infinite value reaches the output."""
    q = torch.zeros(1, 2, 64)
    q[..., 0] = 1
    k, v = torch.zeros(4, 16, 1, 64), torch.ones(4, 16, 1, 64)
    k[1, 2, 0, 0], v[3, 5, 0, 7], v[3, 5, 0, 8] = 40, math.inf, -math.inf
    q, k, v = (x.to(dtype).to(device) for x in (q, k, v))
    table = torch.arange(4, dtype=torch.int32, device=device).view(1, -1)
    out, _ = ops.paged_attention(q, k, v, table, torch.tensor([64], dtype=torch.int32, device=device), 1.0)
    assert (out[0, :, 7] == math.inf).all() and (out[0, :, 8] == -math.inf).all() and (out[0, :, :7] == 1).all()


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("copies,heads", [(40, 1), (1, 3), (1, 20)])
def test_values_that_cancel(ops, device, copies, heads, dtype):
    """Three keys of values 1, -1 and -1 whose weights nearly cancel (1 = a + b but for 2^-11): what is left shows the
    bits that the weights are held in.  The bound: 16 roundings of 32 bits (score, exp, sums, product, quotient) of the
    values' size, 1, and the type's."""
    scores = torch.cat([2.0 ** i * (1 + torch.arange(128, dtype=torch.float64) / 128) for i in (-2, -1, 0)])
    left = 1 - torch.exp(-scores)[:, None] - torch.exp(-scores)
    a, b = torch.nonzero(left.abs() < 2.0 ** -11, as_tuple=True)
    assert len(a) > 50
    a, b = a.repeat(copies), b.repeat(copies)
    B = len(a)
    k, v = torch.zeros(B, 16, 1, 64), torch.zeros(B, 16, 1, 64)
    k[:, 1, 0, 0], k[:, 2, 0, 0] = -scores[a].float(), -scores[b].float()
    v[:, 0], v[:, 1:3] = 1, -1
    q = torch.zeros(B, heads, 64)
    q[..., 0] = 1
    table, lengths = torch.arange(B).int().view(B, 1), torch.full((B,), 3, dtype=torch.int32)
    q, k, v = (x.to(dtype).to(device) for x in (q, k, v))
    out, _ = ops.paged_attention(q, k, v, table.to(device), lengths.to(device), 1.0)
    want = (left[a, b] / (2 - left[a, b]))[:, None, None].expand(B, heads, 64)
    bound = 16 * 2.0 ** -24 + ref.ROUND[dtype] * want.abs() + ref.TINY[dtype]
    off = (out.cpu().double() - want).abs()
    assert (off <= bound).all(), f"{(off / bound).max():.3g} of its bound"
