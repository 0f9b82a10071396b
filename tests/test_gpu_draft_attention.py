"""draft_attention against a plain implementation in 64 bits, node by node."""
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


def make(device, B, S, heads, kv_heads, d, page, longest, dtype, lengths=None, drafted=None, tree=True, seed=0,
         slot_major=False):
    """A batch with its own distinct pages in no order; what no row holds is NaN."""
    g = torch.Generator(device=device).manual_seed(seed)
    rand = lambda *s: torch.randn(*s, generator=g, device=device)  # noqa: E731
    if lengths is None:
        lengths = [max(0, longest - 37 * i * longest // (40 * max(B - 1, 1))) for i in range(B)]
    if drafted is None:
        drafted = [max(0, S - i % 3 * (S // 3)) for i in range(B)]
    width = max(1, -(-longest // page))
    counts = [-(-min(max(n, 0), width * page) // page) for n in lengths]
    pages = sum(counts) + 3
    order = torch.randperm(pages, generator=g, device=device).tolist()
    table = torch.full((B, width), -1, dtype=torch.int32)
    for b, n in enumerate(counts):
        table[b, :n] = torch.tensor([order.pop() for _ in range(n)], dtype=torch.int32)

    def cache():
        if slot_major:
            c = rand(pages, page, kv_heads, d).to(dtype)
        else:
            c = rand(pages, kv_heads, page, d).to(dtype).transpose(1, 2)
        held = torch.zeros(pages, page, dtype=torch.bool)
        for b, n in enumerate(lengths):
            for t in range(min(max(n, 0), width * page)):
                held[table[b, t // page], t % page] = True
        c[~held.to(device)] = math.nan
        return c

    parents = None
    if tree:
        near = torch.rand((B, S), generator=g, device=device) ** 2
        node = torch.arange(S, device=device)
        parents = torch.where(node > 0, (near * node).long().clamp(max=S), -1).int()
        parents = torch.minimum(parents, node.int() - 1)
    i32 = dict(dtype=torch.int32, device=device)
    return dict(q=(2 * rand(B, S, heads, d)).to(dtype), k_cache=cache(), v_cache=cache(), page_table=table.to(device),
                lengths=torch.tensor(lengths, **i32), drafted=torch.tensor(drafted, **i32), parents=parents)


def check(ops, a, scale=None, window=0):
    out, lse = ops.draft_attention(*a.values(), scale, window)
    want, want_lse, bound, lse_bound = ref.draft_attention(
        **{{"page_table": "table"}.get(k, k): v for k, v in a.items()},
        scale=a["q"].shape[-1] ** -0.5 if scale is None else scale, window=window)
    out, lse = out.cpu().double(), lse.cpu().double()
    assert torch.isfinite(out).all()
    bad = (out - want).abs() > bound
    assert not bad.any(), (f"{int(bad.sum())} of {bad.numel()} outputs, first at {bad.nonzero()[0].tolist()}, "
                           f"worst {float(((out - want).abs() / bound).max())} bounds")
    none = want_lse == -math.inf
    assert torch.equal(none, lse == -math.inf)
    assert torch.equal(out[none], torch.zeros_like(out[none]))
    off = (torch.where(none, 0, lse) - torch.where(none, 0, want_lse)).abs()
    assert (off <= lse_bound).all(), float((off / lse_bound.clamp(min=1e-30)).max())
    return out, lse


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("d", [32, 64, 80, 96, 112, 128, 160, 192, 256])
@pytest.mark.parametrize("S,heads,kv_heads", [(3, 8, 2), (12, 8, 2), (25, 4, 1), (37, 8, 2)])
def test_head_sizes_and_rows(ops, device, dtype, d, S, heads, kv_heads):
    """12, 48, 100 and 148 rows of a kv head: each layout, and more than one block."""
    check(ops, make(device, 3, S, heads, kv_heads, d, 16, 200, dtype))


@pytest.mark.parametrize("tree", [True, False])
@pytest.mark.parametrize("page", [1, 7, 16, 64, 200])
@pytest.mark.parametrize("S,longest", [(1, 1), (1, 130), (5, 5), (9, 64), (33, 33), (40, 257), (130, 301)])
def test_lengths_and_pages(ops, device, tree, page, S, longest):
    check(ops, make(device, 4, S, 4, 2, 64, page, longest, BF16, tree=tree, seed=S))


@pytest.mark.parametrize("tree", [True, False])
@pytest.mark.parametrize("window", [1, 2, 5, 31, 64, 100, 1000, 2 ** 40])
@pytest.mark.parametrize("S", [6, 40])
def test_windows(ops, device, tree, window, S):
    check(ops, make(device, 3, S, 6, 2, 64, 8, 150, F16, tree=tree, seed=window % 7), window=window)


@pytest.mark.parametrize("lengths,drafted", [([0, -3, 5, 10 ** 9], [4, 4, 9, 3]), ([7, 8, 9, 50], [0, -1, 8, 10 ** 6]),
                                             ([1, 2, 3, 4], [1, 1, 1, 1])])
@pytest.mark.parametrize("tree", [True, False])
def test_rows_of_no_and_few_tokens(ops, device, lengths, drafted, tree):
    check(ops, make(device, 4, 8, 8, 2, 64, 4, 50, BF16, lengths=lengths, drafted=drafted, tree=tree))


def test_large_trees(ops, device):
    a = make(device, 2, 256, 4, 4, 64, 16, 700, BF16, drafted=[256, 201])
    check(ops, a)
    check(ops, a, window=4)
    a["parents"] = torch.arange(-1, 255, dtype=torch.int32, device=device).expand(2, 256).contiguous()
    one = check(ops, a)
    a["parents"] = None
    assert torch.equal(one[0], check(ops, a)[0])  # the same tiles in the same order


def test_chains_of_any_length(ops, device):
    check(ops, make(device, 2, 700, 2, 1, 64, 16, 900, F16, lengths=[900, 700], drafted=[700, 700], tree=False))
    check(ops, make(device, 1, 400, 16, 2, 32, 16, 400, BF16, tree=False), window=90)


def test_parents_that_are_none(ops, device):
    """What is not a node in front of the node hangs it under the context."""
    a = make(device, 2, 9, 4, 2, 64, 16, 60, BF16, drafted=[9, 5])
    a["parents"] = torch.tensor([[0, 0, 2, 7, -5, 4, 5, 100, 2 ** 31 - 1], [-1, 1, 1, 2, 4, 3, 2, 1, 0]],
                                dtype=torch.int32, device=device)
    check(ops, a)


@pytest.mark.parametrize("S", [4, 20, 40])
def test_holes(ops, device, S):
    """Pages outside the cache are not seen, among the new tokens too; a row of holes only has no output."""
    a = make(device, 4, S, 8, 2, 64, 4, 120, F16, lengths=[120, 90, 60, 44])
    a["page_table"][0, 3] = -1
    a["page_table"][0, 29] = 10 ** 6
    a["page_table"][1, ::2] = -7
    a["page_table"][2] = -1
    check(ops, a)


@pytest.mark.parametrize("slot_major", [False, True])
def test_views_of_one_projection(ops, device, slot_major):
    """q as a view of a fused projection's output; slots or heads as a cache's inner order; odd batch strides."""
    a = make(device, 3, 10, 8, 2, 96, 16, 100, BF16, slot_major=slot_major)
    fused = torch.zeros(3, 11, 12 * 96 + 8, dtype=BF16, device=device)
    q = fused[:, :10, 8:8 + 8 * 96].view(3, 10, 8, 96)
    q.copy_(a["q"])
    a["q"] = q
    want = check(ops, a)
    a["q"] = q.contiguous()
    assert torch.equal(want[0], check(ops, a)[0])


@pytest.mark.parametrize("scale", [0.0, -0.3, 5.0, 1e-6])
def test_scales(ops, device, scale):
    check(ops, make(device, 2, 12, 4, 1, 64, 16, 90, BF16), scale=scale)


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("S", [4, 24, 60])
def test_what_is_not_seen_may_be_anything(ops, device, dtype, S):
    """NaN and infinities in drafted tokens that other branches do not see, and in front of a window."""
    a = make(device, 2, S, 4, 2, 64, 16, 150, dtype, lengths=[150, 150], drafted=[S, S], seed=3)
    want = check(ops, a, window=30)
    b = {k: v.clone() if v is not None else None for k, v in a.items()}
    for row in range(2):
        c = 150 - S
        # The last node is nobody's ancestor: what it holds reaches its own output only.
        t = 150 - 1
        g, s = int(b["page_table"][row, t // 16]), t % 16
        b["k_cache"][g, s], b["v_cache"][g, s] = math.nan, math.inf
        for t in range(0, c - 30):  # in front of every window
            g, s = int(b["page_table"][row, t // 16]), t % 16
            b["k_cache"][g, s], b["v_cache"][g, s] = math.inf, math.nan
    out, lse = ops.draft_attention(*b.values(), None, 30)
    out, lse = out.cpu().double(), lse.cpu().double()
    assert torch.equal(out[:, :-1], want[0][:, :-1]) and torch.equal(lse[:, :-1], want[1][:, :-1])
    assert torch.isnan(out[:, -1]).all()


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("S", [4, 24, 60, 140])
def test_infinite_values_that_are_seen(ops, device, dtype, S):
    """An infinite value is infinite in the outputs of the nodes that see it, at its dimension, and nowhere else:
    in the context, whose weight may be as good as 0, and in a drafted token."""
    a = make(device, 2, S, 4, 2, 64, 16, 400, dtype, lengths=[400, 399], drafted=[S, S], seed=5)
    plain = check(ops, a)
    v = a["v_cache"]
    at = lambda row, t: (int(a["page_table"][row, t // 16]), t % 16)  # noqa: E731
    v[at(0, 5)][0, 3] = math.inf
    v[at(0, 200)][1, 7] = -math.inf
    node = S // 2
    v[at(1, 399 - S + node)][1, 9] = math.inf
    a["q"][0, 0, 0] *= 100  # (a weight that underflows)
    out, lse = ops.draft_attention(*a.values(), None, 0)
    out = out.cpu().double()
    assert (out[0, :, :2, 3] == math.inf).all() and (out[0, :, 2:, 7] == -math.inf).all()
    sees = torch.tensor([node in p for p in ref.paths(a["parents"][1].tolist(), S)])
    assert (out[1, sees][:, 2:, 9] == math.inf).all()
    other = torch.ones_like(out, dtype=torch.bool)
    other[0, :, :2, 3] = other[0, :, 2:, 7] = False
    other[0, 0, 0] = False
    other[1, :, 2:, 9] &= ~sees[:, None]
    assert torch.isfinite(out[other]).all()
    # (in a pass that sets such values apart a part's sums are the same)
    assert ((out - plain[0]).abs()[other] <= 2.0 ** -8 * plain[0].abs()[other] + 2.0 ** -12).all()


def test_extreme_scores(ops, device):
    """One key far above the others, and scores of 10^4."""
    a = make(device, 2, 8, 4, 1, 64, 16, 300, BF16, lengths=[300, 300])
    g = int(a["page_table"][0, 2])
    a["k_cache"][g, 5] *= 30
    check(ops, a)
    check(ops, a, scale=60.0)


@pytest.mark.parametrize("S", [2, 16, 40, 100])
def test_the_same_bits_again(ops, device, S):
    a = make(device, 5, S, 8, 2, 128, 16, 3000, BF16)
    first = ops.draft_attention(*a.values())
    for _ in range(3):
        again = ops.draft_attention(*a.values())
        assert torch.equal(first[0], again[0]) and torch.equal(first[1], again[1])


@pytest.mark.parametrize("B,S,longest", [(1, 4, 5000), (1, 20, 5000), (2, 60, 2500), (70, 3, 120), (130, 2, 20)])
def test_long_rows_and_many(ops, device, B, S, longest):
    check(ops, make(device, B, S, 4, 1, 64, 32, longest, BF16, tree=B % 2 == 1))


def test_one_token_is_paged_attention(ops, device):
    """One new token a row: within both operators' roundings of the operator of single tokens."""
    a = make(device, 6, 1, 8, 2, 128, 16, 500, BF16, drafted=[1] * 6)
    out, lse = ops.draft_attention(*a.values())
    want, want_lse = ops.paged_attention(a["q"][:, 0], a["k_cache"], a["v_cache"], a["page_table"], a["lengths"])
    assert ((out[:, 0].double() - want.double()).abs() <= 2.0 ** -7 * want.double().abs() + 2.0 ** -14).all()
    assert ((lse[:, 0] - want_lse).abs() <= 1e-5).all()


def test_a_graph_and_its_replays(pkg, device):
    """A captured launch reads lengths, tables and parents anew at each replay."""
    a = make(device, 4, 12, 8, 2, 64, 16, 600, BF16)
    op = pkg.DraftAttentionOp(**a)
    op.launch()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        op.launch()
    for n in (600, 77, 12, 5, 300):
        a["lengths"].fill_(n)
        a["drafted"].fill_(min(12, n))
        a["page_table"].copy_(torch.arange(4 * a["page_table"].shape[1], device=device).view(4, -1)
                              % a["k_cache"].shape[0])
        eager = pkg.DraftAttentionOp(**a)
        eager.launch()
        torch.cuda.synchronize()
        want = eager.out.clone(), eager.lse.clone()
        op.out.zero_()
        graph.replay()
        torch.cuda.synchronize()
        same = lambda x, y: torch.equal(torch.nan_to_num(x, 7.0), torch.nan_to_num(y, 7.0))  # noqa: E731
        assert same(op.out, want[0]) and same(op.lse, want[1])


def test_other_streams(ops, device):
    a = make(device, 2, 12, 8, 2, 64, 16, 300, BF16)
    want = ops.draft_attention(*a.values())
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(3)]
    got = []
    for s in streams:
        with torch.cuda.stream(s):
            got.append([ops.draft_attention(*a.values()) for _ in range(4)])
    torch.cuda.synchronize()
    assert all(torch.equal(x, want[0]) and torch.equal(y, want[1]) for run in got for x, y in run)


def test_outputs_of_other_orders(pkg, device):
    """out as a view: what lies beside it stays; no lse."""
    a = make(device, 2, 7, 4, 2, 64, 16, 100, BF16)
    op = pkg.DraftAttentionOp(**a)
    op.launch()
    room = torch.full((2, 9, 6, 64 + 8), 3.0, dtype=BF16, device=device)
    view = room[:, 1:8, 1:5, :64]
    other = pkg.DraftAttentionOp(**a, out=view, lse=False)
    other.launch()
    torch.cuda.synchronize()
    assert torch.equal(view, op.out)
    view.fill_(3.0)
    assert bool((room == 3.0).all())


def test_offsets_beyond_31_bits(ops, device):
    """A cache of more than 2^31 elements, of which the pages in use lie at both ends."""
    pages, page, kv_heads, d = 2 ** 31 // (16 * 2 * 64) + 70, 16, 2, 64
    a = make(device, 2, 10, 4, kv_heads, d, page, 300, BF16)
    small = a["k_cache"].shape[0]
    to = torch.cat((torch.arange(small // 2), torch.arange(pages - (small - small // 2), pages))).to(device)
    for key in ("k_cache", "v_cache"):
        big = torch.zeros(pages, page, kv_heads, d, dtype=BF16, device=device)
        big[to] = a[key]
        a[key + "_big"] = big
    table = a["page_table"].long()
    moved = torch.where(table >= 0, to[table.clamp(min=0)], -1).int()
    want = ops.draft_attention(*[a[k] for k in ("q", "k_cache", "v_cache", "page_table", "lengths", "drafted", "parents")])
    got = ops.draft_attention(a["q"], a["k_cache_big"], a["v_cache_big"], moved, a["lengths"], a["drafted"], a["parents"])
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("d,S,heads,kv_heads", [(64, 130, 8, 2), (128, 90, 4, 1), (80, 150, 2, 1), (256, 70, 4, 1),
                                                (128, 5, 7, 1), (96, 40, 14, 2), (64, 6, 96, 2)])
@pytest.mark.parametrize("window", [0, 45])
def test_many_rows_and_odd_groups(ops, device, dtype, d, S, heads, kv_heads, window):
    """More than 256 rows of a kv head, with masks of trees and windows; 7 and 48 heads of one."""
    check(ops, make(device, 3, S, heads, kv_heads, d, 16, 260, dtype, seed=d), window=window)


@pytest.mark.parametrize("S", [4, 12, 40, 100])
@pytest.mark.parametrize("page", [4, 32])
def test_caches_of_different_layouts(ops, device, S, page):
    """Keys by slots, values by heads, or spread out: the same bits as from caches that are laid out alike."""
    a = make(device, 3, S, 8, 2, 128, page, 300, BF16)
    want = check(ops, a)
    by_slot = torch.empty(a["k_cache"].shape, dtype=BF16, device=device)
    by_slot.copy_(a["k_cache"])
    room = torch.empty(*a["v_cache"].shape[:3], 136, dtype=BF16, device=device)
    room.fill_(math.nan)
    room[..., :128] = a["v_cache"]
    for k, v in ((by_slot, a["v_cache"]), (a["k_cache"], room[..., :128]), (by_slot, room[..., :128])):
        got = ops.draft_attention(a["q"], k, v, a["page_table"], a["lengths"], a["drafted"], a["parents"])
        assert torch.equal(got[0].cpu().double(), want[0]) and torch.equal(got[1].cpu().double(), want[1])


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("S,heads", [(6, 4), (20, 4), (40, 4), (100, 8)])
def test_a_query_that_is_no_number(ops, device, dtype, S, heads):
    """It reaches its own outputs only, and what lies behind a row's nodes reaches none."""
    a = make(device, 2, S, heads, 2, 64, 16, 300, dtype, drafted=[S, S - 2])
    want, want_lse = check(ops, a)
    a["q"][0, S // 2, 1, 3] = math.nan
    a["q"][0, 1, 0] = math.inf
    a["q"][1, S - 2:] = math.nan
    out, lse = (t.cpu().double() for t in ops.draft_attention(*a.values()))
    own = torch.zeros_like(lse, dtype=torch.bool)
    own[0, S // 2, 1] = own[0, 1, 0] = True
    assert torch.isnan(out[own]).all() and torch.isnan(lse[own]).all()
    assert torch.equal(out[~own], want[~own]) and torch.equal(lse[~own], want_lse[~own])


@pytest.mark.parametrize("S,heads,d", [(3, 4, 128), (9, 2, 64), (30, 2, 32), (70, 1, 64), (290, 1, 64)])
def test_rows_of_very_many_parts(ops, device, S, heads, d):
    """One sequence over all workgroups: more parts than one round of the join takes, and infinite values among them."""
    a = make(device, 1, S, heads, 1, d, 64, 33000, BF16, lengths=[33000], drafted=[S], tree=S <= 256)
    plain, _ = check(ops, a)
    again = ops.draft_attention(*a.values())
    assert torch.equal(again[0].cpu().double(), plain)
    for t, e, value in ((7, 3, math.inf), (20000, 9, -math.inf)):
        a["v_cache"][int(a["page_table"][0, t // 64]), t % 64, 0, e] = value
    out = ops.draft_attention(*a.values())[0].cpu().double()
    assert (out[..., 3] == math.inf).all() and (out[..., 9] == -math.inf).all()
    other = torch.ones(d, dtype=torch.bool)
    other[[3, 9]] = False
    # (in a pass that sets such values apart a part's sums are the same)
    assert ((out - plain)[..., other].abs() <= 2.0 ** -8 * plain[..., other].abs() + 2.0 ** -12).all()
