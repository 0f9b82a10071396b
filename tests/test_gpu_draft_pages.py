"""draft_accept, cache_keep and cache_bounds against plain implementations on the host, exactly."""
from __future__ import annotations

import math
import random

import pytest
import torch

import draft_ref as ref

pytestmark = pytest.mark.gpu
F16, BF16, F32 = torch.float16, torch.bfloat16, torch.float32


@pytest.fixture(scope="module")
def ops(pkg, device):
    pkg.torch_ops()
    return torch.ops.mhcpre


# ---- accept --------------------------------------------------------------------


def check_accept(ops, device, tokens, parents, drafted, chosen, lengths, dtype=torch.int64):
    i32 = dict(dtype=torch.int32, device=device)
    to = lambda x: torch.tensor(x, dtype=dtype, device=device).view(len(drafted), -1)  # noqa: E731
    got = ops.draft_accept(to(tokens), None if parents is None else torch.tensor(parents, **i32),
                           torch.tensor(drafted, **i32), to(chosen), torch.tensor(lengths, **i32))
    want = ref.draft_accept(tokens, parents, drafted, chosen, lengths)
    assert got[2].dtype == dtype
    for name, g, w in zip(("path", "accepted", "next", "lengths"), got, want):
        assert g.tolist() == w, name
    return want


@pytest.mark.parametrize("dtype", [torch.int32, torch.int64])
@pytest.mark.parametrize("B,S,vocab", [(1, 1, 3), (3, 2, 2), (5, 9, 2), (4, 63, 3), (9, 64, 2), (2, 65, 2), (33, 100, 3),
                                       (6, 256, 2), (300, 17, 2)])
@pytest.mark.parametrize("tree", [True, False])
def test_accept(ops, device, dtype, B, S, vocab, tree):
    rng = random.Random(B * 1000 + S)
    for _ in range(3):
        tokens, chosen = ([[rng.randrange(vocab) for _ in range(S)] for _ in range(B)] for _ in range(2))
        parents = [[-1] + [rng.randrange(max(0, i - 9), i) for i in range(1, S)] for _ in range(B)] if tree else None
        drafted = [rng.choice((S, S, rng.randint(-2, S + 2))) for _ in range(B)]
        lengths = [rng.choice((1000, rng.randint(-2, S))) for _ in range(B)]
        check_accept(ops, device, tokens, parents, drafted, chosen, lengths, dtype)


def test_accept_whole_chains(ops, device):
    for S in (1, 5, 64, 200, 256):
        row = [[(7 * i) % 50 for i in range(S)]]
        want = check_accept(ops, device, row, None, [S], [row[0][1:] + [99]], [S + 5])
        assert want[1] == [S] and want[2] == [99]


def test_accept_takes_the_first_of_equal_children(ops, device):
    tokens, chosen = [[1, 5, 5, 6, 5]], [[5, 6, 6, 0, 0]]
    want = check_accept(ops, device, tokens, [[-1, 0, 0, 2, 1]], [5], chosen, [9])
    assert want[0] == [[0, 1, -1, -1, -1]] and want[2] == [6]


def test_accept_parents_that_are_none(ops, device):
    check_accept(ops, device, [[1, 1, 1, 1, 1, 1]], [[0, 1, 7, -9, 2 ** 31 - 1, 0]], [6], [[1] * 6], [9])


def test_accept_tokens_of_all_their_bits(ops, device):
    big = 2 ** 40
    check_accept(ops, device, [[0, 3, big + 3]], [[-1, 0, 0]], [3], [[big + 3, 1, -5]], [9])
    check_accept(ops, device, [[0, -1, -2]], [[-1, 0, 0]], [3], [[-2, 1, -(2 ** 62)]], [9])


def test_accept_of_no_rows_and_no_nodes(ops, device):
    i64 = dict(dtype=torch.int64, device=device)
    i32 = dict(dtype=torch.int32, device=device)
    got = ops.draft_accept(torch.zeros(0, 5, **i64), None, torch.zeros(0, **i32), torch.zeros(0, 5, **i64),
                           torch.zeros(0, **i32))
    assert [tuple(t.shape) for t in got] == [(0, 5), (0,), (0,), (0,)]
    got = ops.draft_accept(torch.zeros(2, 0, **i64), None, torch.ones(2, **i32), torch.zeros(2, 0, **i64),
                           torch.full((2,), 4, **i32))
    assert got[1].tolist() == [0, 0] and got[2].tolist() == [-1, -1] and got[3].tolist() == [4, 4]


# ---- keep ----------------------------------------------------------------------


def caches(device, B, page, kv_heads, d, longest, dtype, slot_major=False, seed=0, count=2):
    g = torch.Generator(device=device).manual_seed(seed)
    width = -(-longest // page)
    pages = B * width + 2
    made = []
    for _ in range(count):
        x = torch.randn(pages, page, kv_heads, d, generator=g, device=device).to(dtype)
        made.append(x if slot_major else x.transpose(1, 2).contiguous().transpose(1, 2))
    table = torch.randperm(pages - 2, generator=g, device=device)[:B * width].view(B, width).int().contiguous()
    return made, table


def check_keep(ops, device, made, table, lengths, drafted, path):
    i32 = dict(dtype=torch.int32, device=device)
    args = table, torch.tensor(lengths, **i32), torch.tensor(drafted, **i32), torch.tensor(path, **i32)
    want = ref.cache_keep(made[0], made[1], *(x.cpu() for x in args))
    ops.cache_keep(made[0], made[1], *args)
    for got, w in zip(made, want):
        assert torch.equal(got.cpu(), w)


@pytest.mark.parametrize("dtype", [F16, BF16, F32])
@pytest.mark.parametrize("slot_major", [False, True])
@pytest.mark.parametrize("B,S,page,kv_heads,d", [(1, 1, 4, 1, 8), (3, 7, 4, 2, 64), (5, 40, 16, 8, 128), (2, 300, 7, 1, 6),
                                                 (2, 600, 64, 3, 40), (4, 9, 1, 2, 33), (2, 12, 16, 64, 256)])
def test_keep(ops, device, dtype, slot_major, B, S, page, kv_heads, d):
    rng = random.Random(S)
    made, table = caches(device, B, page, kv_heads, d, S + 50, dtype, slot_major)
    lengths = [rng.randint(S, S + 50) for _ in range(B)]
    path = []
    for _ in range(B):
        some = sorted(rng.sample(range(S), rng.randint(1, S)))
        path.append(some + [-1] * (S - len(some)))
    path[0] = list(range(S))  # nothing moves
    path[-1] = list(range(1, S)) + [-1]  # every one by one place
    check_keep(ops, device, made, table, lengths, [S] * B, path)


def test_keep_odd_paths_and_rows(ops, device):
    """Paths that end at what is no node or does not ascend; rows without tokens; places in holes."""
    made, table = caches(device, 6, 4, 2, 64, 40, BF16)
    table[4, 6] = -1
    table[5, 8] = 10 ** 6
    path = [[0, 2, 1, 5, -1, -1, -1, -1], [1, 3, 9, 4, -1, -1, -1, -1], [-1, 3, 4, 5, 6, 7, -1, -1],
            [2, 4, 6, 7, -1, -1, -1, -1], [1, 2, 3, 4, 5, 6, 7, -1], [3, 4, 5, 6, 7, -1, -1, -1]]
    check_keep(ops, device, made, table, [30, 20, 33, 5, 31, 39], [8, 4, 8, 8, 8, 8], path)
    check_keep(ops, device, made, table, [0, -5, 10 ** 9, 30, 31, 39], [8, 8, 8, -1, 0, 10 ** 9], path)


def test_keep_of_other_orders(ops, device):
    """Views of wider caches, and caches that 16-byte pieces do not fit."""
    for d, off in ((64, 0), (64, 8), (64, 1), (20, 3)):
        made, table = caches(device, 2, 4, 2, d, 40, F16)
        wide = [torch.zeros(x.shape[0], 4, 3, d + 16, dtype=F16, device=device) for x in made]
        views = [w[:, :, 1:, off:off + d] for w in wide]
        for v, x in zip(views, made):
            v.copy_(x)
        path = [[0, 2, 5, 6, -1, -1, -1, -1], [3, 4, 5, 7, -1, -1, -1, -1]]
        check_keep(ops, device, views, table, [30, 22], [8, 8], path)
        for w, v in zip(wide, views):
            v.zero_()
            assert not w.any()


# ---- bounds --------------------------------------------------------------------


def check_bounds(ops, device, k, lo, hi, table, lengths, counts, tokens):
    i32 = dict(dtype=torch.int32, device=device)
    args = table, torch.tensor(lengths, **i32), torch.tensor(counts, **i32)
    want = ref.cache_bounds(k, *(x.cpu() for x in args), lo, hi, tokens)
    ops.cache_bounds(k, *args, lo, hi, tokens)
    nan = torch.isnan(want[0]) | torch.isnan(want[1])
    for got, w in zip((lo, hi), want):
        got = got.cpu().double()
        assert torch.equal(torch.isnan(got), nan)
        assert torch.equal(torch.where(nan, 0, got), torch.where(nan, 0, w))


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("d", [32, 64, 80, 96, 112, 128, 160, 192, 256])
@pytest.mark.parametrize("page", [1, 7, 16, 100])
def test_bounds(ops, device, dtype, d, page):
    (k, lo, hi), table = caches(device, 4, page, 3, d, 230, dtype, count=3, slot_major=page % 2 == 0)
    lo, hi = (x[:, 0].clone() for x in (lo.contiguous(), hi.contiguous()))
    check_bounds(ops, device, k, lo, hi, table, [230, 100, 64, 1], [230, 100, 64, 1], 230)  # anew
    check_bounds(ops, device, k, lo, hi, table, [229, 101, 70, 2], [1, 1, 1, 1], 1)  # a step
    check_bounds(ops, device, k, lo, hi, table, [0, 150, 10 ** 9, -3], [5, 49, 10 ** 9, 7], 60)  # a chunk; clamped


def test_bounds_holes_and_rows(ops, device):
    (k, lo, hi), table = caches(device, 3, 8, 2, 64, 90, BF16, count=3)
    lo, hi = (x[:, 0].clone() for x in (lo.contiguous(), hi.contiguous()))
    table[0, 2], table[1, 0], table[2] = -1, 10 ** 6, -1
    check_bounds(ops, device, k, lo, hi, table, [90, 50, 60], [90, -4, 60], 90)
    check_bounds(ops, device, k, lo, hi, table, [90, 50, 60], [0, 50, 0], 0)


@pytest.mark.parametrize("dtype", [F16, BF16])
def test_bounds_of_exceptional_keys(ops, device, dtype):
    """Infinities, both zeros, NaN of both signs, the smallest values; NaN in old bounds; NaN behind the row's end."""
    (k, lo, hi), table = caches(device, 1, 8, 1, 64, 32, dtype, count=3)
    lo, hi = (x[:, 0].clone() for x in (lo.contiguous(), hi.contiguous()))
    at = [int(g) for g in table[0]]
    k[at[0], 2, 0, 0], k[at[0], 3, 0, 0], k[at[0], 4, 0, 1] = math.inf, -math.inf, math.nan
    bits = k.view(torch.int16)
    bits[at[0], 5, 0, 2] = -1  # a NaN below 0
    k[at[1], :, 0, 3] = 0.0
    k[at[1], 1, 0, 3] = -0.0
    bits[at[1], 2, 0, 4], bits[at[1], 3, 0, 4] = 1, -32767  # the smallest of both signs
    k[at[2], 6:, 0] = math.nan
    check_bounds(ops, device, k, lo, hi, table, [22], [22], 22)
    assert lo[at[1], 0, 3].view(torch.int16).item() == -32768 and hi[at[1], 0, 3].view(torch.int16).item() == 0
    lo[at[2], 0, 5] = math.nan
    k[at[2], 6, 0] = 1.0
    check_bounds(ops, device, k, lo, hi, table, [23], [1], 1)


def test_bounds_of_other_orders(ops, device):
    (k, lo, hi), table = caches(device, 2, 8, 2, 64, 40, BF16, count=3)
    room = torch.full((2, k.shape[0], 4, 72), 5.0, dtype=BF16, device=device)
    lo_v, hi_v = room[0, :, 1:3, 8:], room[1, :, ::2, :64]
    lo_v.copy_(lo[:, 0])
    hi_v.copy_(hi[:, 0])
    check_bounds(ops, device, k, lo_v, hi_v, table, [40, 31], [9, 31], 31)
    lo_v.fill_(5.0)
    hi_v.fill_(5.0)
    assert bool((room == 5.0).all())


def test_bounds_go_with_their_pages(ops, device):
    """cache_copy_pages copies bounds as caches with pages of one slot."""
    (k, lo, hi), table = caches(device, 1, 8, 2, 64, 40, BF16, count=3)
    lo, hi = (x[:, 0].clone() for x in (lo.contiguous(), hi.contiguous()))
    src, dst = (torch.tensor(x, dtype=torch.int32, device=device) for x in ([0, 3], [5, 4]))
    ops.cache_copy_pages(lo[:, None], hi[:, None], src, dst)
    assert torch.equal(lo[5], lo[0]) and torch.equal(hi[4], hi[3])


def test_graphs_of_the_three(pkg, device):
    """Captured together, replayed on new contents."""
    i32 = dict(dtype=torch.int32, device=device)
    (k, v, lo, hi), table = caches(device, 3, 8, 2, 64, 60, BF16, count=4)
    lo, hi = (x[:, 0].clone() for x in (lo.contiguous(), hi.contiguous()))
    lengths, drafted, counts = torch.full((3,), 50, **i32), torch.full((3,), 9, **i32), torch.zeros(3, **i32)
    tokens, chosen = torch.zeros(3, 9, dtype=torch.int64, device=device), torch.zeros(3, 9, dtype=torch.int64, device=device)
    parents = torch.zeros(3, 9, **i32)
    accept = pkg.DraftAcceptOp(tokens, parents, drafted, chosen, lengths)
    keep = pkg.CacheKeepOp(k, v, table, lengths, drafted, accept.path)
    bounds = pkg.CacheBoundsOp(k, table, accept.new_lengths, accept.accepted, lo, hi, 9)
    for op in (accept, keep, bounds):
        op.launch()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        for op in (accept, keep, bounds):
            op.launch()
    g = torch.Generator(device=device).manual_seed(1)
    for n in (60, 9, 33, 47):
        for x in (k, v, lo, hi):
            x.copy_(torch.randn(x.shape, generator=g, device=device))
        lengths.fill_(n)
        tokens.copy_(torch.randint(0, 2, (3, 9), generator=g, device=device))
        chosen.copy_(torch.randint(0, 2, (3, 9), generator=g, device=device))
        parents.copy_((torch.rand((3, 9), generator=g, device=device) * torch.arange(9, device=device)).int() - 0)
        want = ref.draft_accept(tokens.tolist(), parents.tolist(), drafted.tolist(), chosen.tolist(), lengths.tolist())
        path, accepted, new = (torch.tensor(want[x], dtype=torch.int32) for x in (0, 1, 3))
        want_k, want_v = ref.cache_keep(k, v, table.cpu(), lengths.cpu(), drafted.cpu(), path)
        want_lo, want_hi = ref.cache_bounds(want_k, table.cpu(), new, accepted, lo, hi, 9)
        graph.replay()
        torch.cuda.synchronize()
        assert accept.path.tolist() == want[0] and accept.next.tolist() == want[2]
        assert torch.equal(k.cpu(), want_k) and torch.equal(v.cpu(), want_v)
        assert torch.equal(lo.cpu().double(), want_lo) and torch.equal(hi.cpu().double(), want_hi)
