"""sparse_attention against a plain implementation in 64 bits: the columns exactly, outputs within derived bounds."""
from __future__ import annotations

import math

import pytest
import torch

import draft_ref as ref

pytestmark = pytest.mark.gpu
F16, BF16 = torch.float16, torch.bfloat16


@pytest.fixture(scope="module")
def ops(pkg, device):
    pkg.torch_ops()
    return torch.ops.mhcpre


def make(device, B, heads, kv_heads, d, page, longest, dtype, lengths=None, seed=0, slot_major=False):
    """Rows of distinct pages with their keys' bounds; what no row holds is NaN."""
    g = torch.Generator(device=device).manual_seed(seed)
    rand = lambda *s: torch.randn(*s, generator=g, device=device)  # noqa: E731
    if lengths is None:
        lengths = [max(0, longest - 39 * i * longest // (40 * max(B - 1, 1))) for i in range(B)]
    width = max(1, -(-longest // page))
    counts = [-(-min(max(n, 0), width * page) // page) for n in lengths]
    pages = sum(counts) + 3
    order = torch.randperm(pages, generator=g, device=device).tolist()
    table = torch.full((B, width), -1, dtype=torch.int32)
    for b, n in enumerate(counts):
        table[b, :n] = torch.tensor([order.pop() for _ in range(n)], dtype=torch.int32)
    k = rand(pages, kv_heads, page, d) + rand(pages, kv_heads, 1, d)
    v = rand(pages, kv_heads, page, d)
    k, v = (x.to(dtype).transpose(1, 2) for x in (k, v))
    if slot_major:
        k, v = k.contiguous(), v.contiguous()
    held = torch.zeros(pages, page, dtype=torch.bool)
    for b, n in enumerate(lengths):
        for t in range(min(max(n, 0), width * page)):
            held[table[b, t // page], t % page] = True
    held = held.to(device)
    k[~held], v[~held] = math.nan, math.nan
    there = held[..., None, None]
    lo, hi = torch.where(there, k, math.inf).amin(1), torch.where(there, k, -math.inf).amax(1)
    return dict(q=(2 * rand(B, heads, d)).to(dtype), k_cache=k, v_cache=v, lo=lo, hi=hi, table=table.to(device),
                lengths=torch.tensor(lengths, dtype=torch.int32, device=device))


def check(ops, a, top, first=1, last=1, scale=None):
    out, lse, columns = ops.sparse_attention(*a.values(), top, first, last, scale)
    want, want_lse, bound, lse_bound, want_columns = ref.sparse_attention(
        **a, top=top, first=first, last=last, scale=a["q"].shape[-1] ** -0.5 if scale is None else scale)
    assert torch.equal(columns.cpu(), want_columns)
    out, lse = out.cpu().double(), lse.cpu().double()
    assert torch.isfinite(out).all()
    bad = (out - want).abs() > bound
    assert not bad.any(), (int(bad.sum()), float(((out - want).abs() / bound).max()))
    none = want_lse == -math.inf
    assert torch.equal(none, lse == -math.inf) and torch.equal(out[none], torch.zeros_like(out[none]))
    off = (torch.where(none, 0, lse) - torch.where(none, 0, want_lse)).abs()
    assert (off <= lse_bound).all()
    return out, lse, columns


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("d", [32, 64, 80, 96, 112, 128, 160, 192, 256])
@pytest.mark.parametrize("heads,kv_heads", [(8, 2), (3, 3), (20, 1)])
def test_head_sizes(ops, device, dtype, d, heads, kv_heads):
    check(ops, make(device, 3, heads, kv_heads, d, 16, 700, dtype), 9)


@pytest.mark.parametrize("page", [1, 7, 16, 64])
@pytest.mark.parametrize("longest", [1, 5, 64, 130, 1000])
@pytest.mark.parametrize("top,first,last", [(1, 0, 0), (1, 1, 0), (2, 1, 1), (5, 0, 2), (9, 4, 5), (40, 2, 3),
                                            (2000, 1, 1)])
def test_lengths_pages_and_counts(ops, device, page, longest, top, first, last):
    check(ops, make(device, 4, 4, 2, 64, page, longest, BF16, seed=top), top, first, last)


def test_rows_of_no_and_few_tokens(ops, device):
    a = make(device, 6, 4, 2, 64, 8, 100, F16, lengths=[0, -4, 1, 8, 9, 10 ** 9])
    check(ops, a, 4)
    check(ops, a, 4, 0, 0)


def test_holes(ops, device):
    a = make(device, 4, 8, 2, 64, 8, 200, BF16, lengths=[200, 180, 90, 77])
    a["table"][0, ::3] = -1
    a["table"][1, 0] = 10 ** 6
    a["table"][1, 22] = -5  # the last column
    a["table"][2] = -1
    for top, first, last in ((5, 1, 1), (6, 3, 3), (20, 0, 0)):
        check(ops, a, top, first, last)


def test_equal_scores_go_to_the_lower_column(ops, device):
    """Pages with equal bounds, and scores of 0 of both signs."""
    a = make(device, 2, 4, 2, 64, 4, 400, F16)
    a["lo"].fill_(-1.0)
    a["hi"].fill_(2.0)
    out, lse, columns = check(ops, a, 7, 1, 1)
    assert columns[0, 0].tolist() == [0, 1, 2, 3, 4, 5, 99]
    a["lo"].zero_()
    a["hi"].zero_()
    a["hi"][::2] = -0.0
    check(ops, a, 7, 0, 0)
    # Two kinds of pages: all of the better one, the first of the other.
    better = a["table"][0, 10:60:10].long()
    a["hi"].fill_(1.0)
    a["lo"].fill_(1.0)
    a["q"].fill_(1.0)
    a["hi"][better] = 1.5
    a["lo"][better] = 1.5
    columns = check(ops, a, 9, 0, 0)[2]
    assert columns[0, 0].tolist() == [0, 1, 2, 3, 10, 20, 30, 40, 50]


def test_scores_that_differ_in_their_last_bits(ops, device):
    """Sums whose 24 bits agree: the order is that of 64 bits."""
    a = make(device, 1, 2, 1, 64, 1, 500, BF16)
    a["q"].fill_(1.0)
    tiny = (torch.randperm(a["lo"].shape[0], device=device).float() * 2.0 ** -30).to(BF16)
    for x in ("lo", "hi"):
        x = a[x]
        x.fill_(1.0)
        x[:, 0, 0] = 256.0
        x[:, 0, 1] = tiny
    for top in (1, 17, 250):
        check(ops, a, top, 0, 0)


def test_exceptional_bounds(ops, device):
    """A NaN score is above all others, infinite ones above and below the finite."""
    a = make(device, 1, 2, 1, 64, 4, 200, F16, lengths=[200])
    page = lambda c: int(a["table"][0, c])  # noqa: E731
    a["q"][0, :, 0], a["q"][0, :, 1] = 1.0, -1.0
    a["hi"][page(20), 0, 0] = math.nan
    a["hi"][page(30), 0, 0] = math.inf
    a["hi"][page(40), 0, 0] = -math.inf
    a["lo"][page(35), 0, 1] = -math.inf
    taken = lambda top: check(ops, a, top, 0, 0)[2][0, 0].tolist()  # noqa: E731
    assert taken(1) == [20] and taken(3) == [20, 30, 35]
    assert 40 not in taken(49) and taken(50) == list(range(50))


@pytest.mark.parametrize("top", [5, 300, 1025])
def test_many_columns(ops, device, top):
    """More columns than a workgroup's threads, several rounds of every loop."""
    check(ops, make(device, 2, 4, 1, 32, 1, 5000, BF16, lengths=[5000, 4097]), top, 2, 3)


def test_ties_beyond_one_round(ops, device):
    a = make(device, 1, 2, 1, 32, 1, 3000, F16, lengths=[3000])
    a["lo"].fill_(0.5)
    a["hi"].fill_(0.5)
    columns = check(ops, a, 1500, 0, 1)[2]
    assert columns[0, 0].tolist() == list(range(1499)) + [2999]


def test_bounds_hold(ops, device):
    """With all pages taken it is paged attention, whatever the bounds."""
    a = make(device, 5, 8, 2, 128, 16, 600, BF16)
    got = ops.sparse_attention(*a.values(), 38)
    want = ops.paged_attention(a["q"], a["k_cache"], a["v_cache"], a["table"], a["lengths"])
    assert ((got[0].double() - want[0].double()).abs() <= 2.0 ** -7 * want[0].double().abs() + 2.0 ** -14).all()
    assert ((got[1] - want[1]).abs() <= 1e-5).all()


def test_views_and_other_orders(ops, pkg, device):
    a = make(device, 3, 4, 2, 64, 8, 150, BF16, slot_major=True)
    want = check(ops, a, 6)
    fused = torch.zeros(3, 8 * 64 + 16, dtype=BF16, device=device)
    q = fused[:, 16:16 + 4 * 64].view(3, 4, 64)
    q.copy_(a["q"])
    room = torch.zeros(2, a["lo"].shape[0], 4, 72, dtype=BF16, device=device)
    lo, hi = room[0, :, 1:3, 8:], room[1, :, ::2, :64]
    lo.copy_(a["lo"])
    hi.copy_(a["hi"])
    b = {**a, "q": q, "lo": lo, "hi": hi}
    got = check(ops, b, 6)
    assert all(torch.equal(x, y) for x, y in zip(got, want))
    out = torch.full((3, 6, 80), 3.0, dtype=BF16, device=device)
    op = pkg.SparseAttentionOp(*b.values(), 6, out=out[:, 1:5, 8:72], lse=False)
    op.launch()
    torch.cuda.synchronize()
    assert torch.equal(out[:, 1:5, 8:72].cpu().double(), want[0])
    out[:, 1:5, 8:72] = 3.0
    assert bool((out == 3.0).all())


def test_leading_dimensions(ops, device):
    a = make(device, 6, 4, 2, 64, 8, 150, BF16)
    want = ops.sparse_attention(*a.values(), 5)
    a["q"] = a["q"].view(2, 3, 4, 64)
    got = ops.sparse_attention(*a.values(), 5)
    assert [tuple(t.shape) for t in got] == [(2, 3, 4, 64), (2, 3, 4), (2, 3, 2, 5)]
    assert all(torch.equal(x.flatten(), y.flatten()) for x, y in zip(got, want))


def test_the_same_bits_again(ops, device):
    a = make(device, 3, 16, 2, 128, 16, 6000, BF16)
    first = ops.sparse_attention(*a.values(), 100)
    for _ in range(3):
        assert all(torch.equal(x, y) for x, y in zip(first, ops.sparse_attention(*a.values(), 100)))


def test_short_rows_in_large_batches(ops, device):
    """Rows that a wave does alone."""
    check(ops, make(device, 160, 8, 4, 64, 4, 60, F16), 5)


def test_a_graph_and_its_replays(pkg, device):
    a = make(device, 4, 8, 2, 64, 8, 700, BF16)
    for x in ("k_cache", "v_cache", "lo", "hi"):
        a[x].copy_(torch.nan_to_num(a[x], 0.5, 1.0, -1.0))
    op = pkg.SparseAttentionOp(*a.values(), 9)
    op.launch()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        op.launch()
    width = a["table"].shape[1]
    for step, n in enumerate((700, 77, 0, 300, 8)):
        a["lengths"].fill_(n)
        a["table"].copy_((torch.arange(4 * width, device=device).view(4, -1) * (2 * step + 1)) % a["lo"].shape[0])
        a["q"].mul_(-1.0)
        eager = pkg.SparseAttentionOp(*a.values(), 9)
        eager.launch()
        torch.cuda.synchronize()
        want = [t.clone() for t in (eager.out, eager.lse, eager.columns)]
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(x, y) for x, y in zip((op.out, op.lse, op.columns), want))


def test_other_streams(ops, device):
    a = make(device, 3, 8, 2, 64, 8, 700, BF16)
    want = ops.sparse_attention(*a.values(), 9)
    torch.cuda.synchronize()
    got = []
    for s in [torch.cuda.Stream() for _ in range(3)]:
        with torch.cuda.stream(s):
            got += [ops.sparse_attention(*a.values(), 9) for _ in range(4)]
    torch.cuda.synchronize()
    assert all(torch.equal(x, y) for run in got for x, y in zip(run, want))


@pytest.mark.parametrize("longest,top", [(2049, 40), (8192, 7), (8193, 500), (20000, 9000)])
def test_tables_of_several_segments(ops, device, longest, top):
    """Columns in registers, and read anew in each round; holes among them."""
    a = make(device, 2, 4, 1, 32, 1, longest, F16, lengths=[longest, longest - 1000])
    a["table"][0, 5::97] = -1
    check(ops, a, top, 2, 3)


def test_ties_over_segments(ops, device):
    a = make(device, 1, 2, 1, 32, 1, 20000, F16, lengths=[20000])
    a["lo"].fill_(0.5)
    a["hi"].fill_(0.5)
    better = int(a["table"][0, 15000])
    a["lo"][better], a["hi"][better] = -8.0, 8.0
    columns = check(ops, a, 9000, 0, 1)[2]
    assert columns[0, 0].tolist() == list(range(8998)) + [15000, 19999]


def test_offsets_beyond_31_bits(ops, device):
    """Bounds and caches of more than 2^31 elements, of which the pages in use lie at both ends: kept, bounded, selected."""
    page, kv_heads, d = 1, 16, 64
    pages = 2 ** 31 // (kv_heads * d) + 50
    a = make(device, 1, 16, kv_heads, d, page, 61, BF16)
    small = a["k_cache"].shape[0]
    to = torch.cat((torch.arange(small // 2), torch.arange(pages - (small - small // 2), pages))).to(device)
    big = {}
    for key in ("k_cache", "v_cache", "lo", "hi"):
        big[key] = torch.zeros(pages, *a[key].shape[1:], dtype=BF16, device=device)
        big[key][to] = a[key]
    table = torch.where(a["table"] >= 0, to[a["table"].long().clamp(min=0)], -1).int()
    i32 = lambda v: torch.tensor(v, dtype=torch.int32, device=device)  # noqa: E731
    path = i32([[0, 3, 5, 8, -1, -1, -1, -1, -1, -1]])
    lengths, drafted, accepted, after = a["lengths"], i32([10]), i32([4]), a["lengths"] - 6
    results = []
    for at, tab in ((a, a["table"]), (big, table)):
        ops.cache_keep(at["k_cache"], at["v_cache"], tab, lengths, drafted, path)
        ops.cache_bounds(at["k_cache"], tab, after, accepted, at["lo"], at["hi"], 10)
        results.append(ops.sparse_attention(a["q"], at["k_cache"], at["v_cache"], at["lo"], at["hi"], tab, after, 20))
    for key in big:
        there = a["table"][0, :int(after)].long()
        assert torch.equal(big[key][table[0, :int(after)].long()], a[key][there])
    assert all(torch.equal(x, y) for x, y in zip(*results))
