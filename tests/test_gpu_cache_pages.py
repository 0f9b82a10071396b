"""cache_update, cache_compact and cache_copy_pages against plain Python."""
from __future__ import annotations

import random

import pytest
import torch

import serve_ref as ref

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ops(pkg, device):
    pkg.torch_ops()
    return torch.ops.mhcpre


def _i32(v, device, shape=None):
    t = torch.tensor(v, dtype=torch.int32, device=device)
    return t if shape is None else t.view(shape)


def _lists(outs):
    return [o.cpu().tolist() for o in outs]


def _state(rng, rows, width, pages, page, share=0.3, holes=0.0):
    """Rows of pages that no two hold, but for the shared beginnings of some."""
    free = list(range(pages))
    rng.shuffle(free)
    table, lengths = [], []
    for r in range(rows):
        n = rng.randint(0, width)
        row, length = [], n * page - rng.randint(0, page - 1) if n else 0
        if r and rng.random() < share:
            other = rng.randrange(r)
            row = table[other][:min(n, -(-lengths[other] // page))]
            if row and rng.random() < 0.7:  # with its partly filled last page
                length = max(0, min(len(row) * page - rng.randint(0, page - 1), lengths[other]))
                n = len(row)
        while len(row) < n and free:
            row = row + [free.pop()]
        length = min(length, len(row) * page)
        row = [-1 if rng.random() < holes else g for g in row]
        stale = [rng.randint(-1, pages - 1) for _ in range(width - len(row))]  # beyond the length: anything
        table.append(row + stale)
        lengths.append(length)
    return table, lengths


def _update(ops, device, table, lengths, parents, counts, pages, page, tokens):
    R, W = len(table), len(table[0])
    got = ops.cache_update(_i32(table, device, (R, W)), _i32(lengths, device), _i32(parents, device),
                           _i32(counts, device), pages, page, tokens)
    want = ref.update(table, lengths, parents, counts, pages, page, tokens)
    for name, g, w in zip(("table", "lengths", "slots", "granted", "src", "dst"), _lists(got), want):
        assert g == list(w), name
    return want


@pytest.mark.parametrize("rows,width,pages,page,tokens", [
    (1, 1, 1, 1, 1), (4, 3, 7, 4, 1), (64, 16, 700, 16, 1), (64, 16, 300, 16, 40), (37, 9, 100, 1, 3),
    (200, 5, 900, 64, 2), (1500, 4, 4000, 8, 5), (3, 700, 1500, 7, 900), (30, 50, 40001, 16, 33),
    (17, 30, 300000, 16, 100), (2500, 40, 70000, 3, 7), (5, 3, 33, 100, 0)])
@pytest.mark.parametrize("seed", [0, 1])
def test_update(ops, device, rows, width, pages, page, tokens, seed):
    rng = random.Random(seed * 1000 + rows)
    table, lengths = _state(rng, rows, width, pages, page, holes=0.02 if seed else 0.0)
    parents = [rng.choice((r, r, r, rng.randrange(rows), -1)) for r in range(rows)]
    counts = [rng.choice((1, 1, 0, tokens, rng.randint(0, max(tokens, 1)))) for _ in range(rows)]
    _update(ops, device, table, lengths, parents, counts, pages, page, tokens)


def test_update_beams_reorder(ops, device):
    """Rows that go on from one another at once, each appending: all get private copies of their last pages."""
    table = [[0, 1, 9, 9], [2, 3, 9, 9], [4, 5, 9, 9]]
    want = _update(ops, device, table, [6, 7, 8], [1, 0, 1], [1, 1, 1], 16, 4, 1)
    assert want[4] == [3, -1, 3] and want[5] == [4, -1, 5]  # row 2's old pages are free at once


def test_update_runs_out(ops, device):
    """Free pages go to the first rows; a row that needs none is served whatever the rows before it asked."""
    table = [[0, -1, -1], [1, -1, -1], [2, -1, -1], [3, -1, -1]]
    want = _update(ops, device, table, [4, 4, 3, 4], [0, 1, 2, 3], [5, 4, 1, 1], 6, 4, 8)
    assert want[3] == [5, 0, 1, 0]
    _update(ops, device, table, [4, 4, 4, 4], [0, 1, 2, 3], [1, 1, 1, 1], 4, 4, 1)  # none is free
    _update(ops, device, table, [12, 9, 4, 4], [0, 1, 2, 3], [1, 1, 1, 1], 40, 4, 1)  # a full row


def test_update_out_of_range(ops, device):
    """Parents, counts, lengths and pages beyond their ranges."""
    table = [[0, 2 ** 31 - 1, -7], [7, 1, 2], [3, 4, 5]]
    _update(ops, device, table, [12, 10 ** 9, -5], [0, 1, 2], [-3, 2, 100], 7, 4, 6)
    _update(ops, device, table, [12, 7, 9], [5, -2 ** 31, 2 ** 31 - 1], [3, 2, 1], 7, 4, 6)
    _update(ops, device, [[-1, -1, -1]], [5], [0], [1], 7, 4, 6)  # appends into a hole


def test_update_empty(ops, device):
    out = ops.cache_update(_i32([], device, (0, 4)), _i32([], device), _i32([], device), _i32([], device), 8, 4, 2)
    assert out[0].shape == (0, 4) and out[2].shape == (0, 2)


@pytest.mark.parametrize("rows,width,pages,page", [(1, 1, 1, 1), (4, 3, 7, 4), (64, 16, 1500, 16), (200, 5, 2001, 64),
                                                   (1500, 4, 4000, 8), (3, 700, 5000, 7), (30, 50, 300001, 16),
                                                   (2500, 40, 70000, 3), (2, 3, 2 ** 20 + 5, 2)])
@pytest.mark.parametrize("seed", [0, 1])
def test_compact(ops, device, rows, width, pages, page, seed):
    rng = random.Random(seed * 1000 + rows)
    table, lengths = _state(rng, rows, width, pages, page, holes=0.05 if seed else 0.0)
    got = ops.cache_compact(_i32(table, device, (rows, width)), _i32(lengths, device), pages, page)
    for name, g, w in zip(("table", "src", "dst", "used"), _lists(got), ref.compact(table, lengths, pages, page)):
        assert g == list(w), name


@pytest.mark.parametrize("pages", [1, 31, 32, 33, 64, 1000])
def test_compact_full_and_empty(ops, device, pages):
    for n in (0, pages):
        table, lengths = [list(range(n)) + [-1] * (pages - n)], [n * 2]
        got = ops.cache_compact(_i32(table, device, (1, pages)), _i32(lengths, device), pages, 2)
        assert _lists(got) == [list(w) for w in ref.compact(table, lengths, pages, 2)]
    got = ops.cache_compact(_i32([], device, (0, 4)), _i32([], device), pages, 2)
    assert got[3].item() == 0 and (got[1] == -1).all()


def _caches(device, pages, page, kv_heads, d, dtype, order, gap):
    """A pair of caches whose memory has (pages, slots, heads) in `order`, rows `gap` elements apart."""
    dims = [(pages, page, kv_heads)[i] for i in order]
    out = []
    for _ in range(2):
        base = torch.randint(-2 ** 15, 2 ** 15, dims + [d + gap], dtype=torch.int16, device=device)
        base = base.to(torch.int32) if dtype == torch.float32 else base
        out.append(base.view(dtype)[..., :d].permute(*[order.index(i) for i in range(3)], 3))
    return out


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16, torch.float32])
@pytest.mark.parametrize("order", [(0, 1, 2), (0, 2, 1), (1, 0, 2), (2, 0, 1)])
@pytest.mark.parametrize("pages,page,kv_heads,d,gap,n", [(40, 16, 8, 128, 0, 19), (9, 7, 3, 80, 0, 4), (9, 1, 1, 2, 0, 4),
                                                         (12, 5, 2, 33, 3, 5), (12, 4, 2, 64, 8, 5),
                                                         (3000, 2, 1, 16, 0, 1400)])
def test_copy_pages(ops, device, pages, page, kv_heads, d, gap, n, order, dtype):
    k, v = _caches(device, pages, page, kv_heads, d, dtype, order, gap)
    whole = [(c, c._base) for c in (k, v)]
    perm = torch.randperm(pages)
    src, dst = perm[:n].int(), perm[n:2 * n].int()
    if n > 4:  # pairs that copy nothing
        src[0], dst[1], src[2], dst[3] = -1, -1, pages, 2 ** 31 - 1
    size = torch.int32 if dtype == torch.float32 else torch.int16
    want = []
    for c, base in whole:
        w = base.clone()
        view = w.as_strided(c.shape, c.stride(), c.storage_offset()).view(size)
        for s, t in zip(src.tolist(), dst.tolist()):
            if 0 <= s < pages and 0 <= t < pages:
                view[t] = view[s].clone()
        want.append(w.view(size))
    ops.cache_copy_pages(k, v, src.to(device), dst.to(device))
    for (c, base), w in zip(whole, want):
        assert torch.equal(base.view(size), w)  # the gaps are as they were, too


def test_copy_beyond_32_bits(ops, device):
    k = torch.zeros(70000, 64, 8, 128, dtype=torch.bfloat16, device=device)
    v = torch.zeros(70000, 64, 8, 128, dtype=torch.bfloat16, device=device)
    k[69999], v[3] = 1, 2
    ops.cache_copy_pages(k, v, _i32([69999, 3], device), _i32([0, 65537], device))
    assert (k[0] == 1).all() and (v[65537] == 2).all() and (v[0] == 0).all() and (k[65537] == 0).all()
    assert int((k != 0).any(-1).any(-1).any(-1).sum()) == 2


def test_a_serving_life(ops, device):
    """Prompts, forks, steps, ends and a compaction: every row's tokens are always where its table says."""
    rng = random.Random(7)
    rows, width, pages, page, tokens = 12, 10, 90, 4, 9
    table = torch.full((rows, width), -1, dtype=torch.int32, device=device)
    lengths = torch.zeros(rows, dtype=torch.int32, device=device)
    k = torch.zeros(pages, page, 1, 2, dtype=torch.float32, device=device)
    v = torch.zeros_like(k)
    told = [[] for _ in range(rows)]
    for step in range(40):
        parents = [rng.choice((r, r, r, r, r, rng.randrange(rows), -1)) for r in range(rows)]
        counts = [rng.choice((1, 1, 1, 0, tokens)) for _ in range(rows)]
        table, lengths, slots, granted, src, dst = ops.cache_update(
            table, lengths, _i32(parents, device), _i32(counts, device), pages, page, tokens)
        ops.cache_copy_pages(k, v, src, dst)
        told = [list(told[p]) if 0 <= p < rows else [] for p in parents]
        for r, n in enumerate(granted.tolist()):
            fresh = [float(step * 1000 + r * 20 + i) for i in range(n)]
            at = slots[r, :n]
            k[at // page, at % page, 0, 0] = torch.tensor(fresh, device=device)
            v[at // page, at % page, 0, 1] = -torch.tensor(fresh, device=device)
            told[r] += fresh
        if step % 7 == 6:
            table, src, dst, used = ops.cache_compact(table, lengths, pages, page)
            ops.cache_copy_pages(k, v, src, dst)
            assert int(table.max()) < int(used)
        for r in range(rows):
            t = torch.arange(len(told[r]), device=device)
            at = table[r].long()[t // page]
            assert lengths[r] == len(told[r])
            assert k[at, t % page, 0, 0].tolist() == told[r]
            assert v[at, t % page, 0, 1].tolist() == [-x for x in told[r]]


def test_streams_workspace_contents_and_graphs(pkg, device):
    rng = random.Random(3)
    table, lengths = _state(rng, 50, 20, 900, 16)
    t, n = _i32(table, device, (50, 20)), _i32(lengths, device)
    parents, counts = _i32(list(range(50)), device), _i32([1] * 50, device)
    up = pkg.CacheUpdateOp(t, n, parents, counts, 900, 16)
    co = pkg.CacheCompactOp(t, n, 900, 16)
    for op in (up, co):
        op.workspace.fill_(255)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    up.launch(side)
    co.launch(side)
    side.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        up.launch()
        co.launch()
    for step in range(4):
        graph.replay()
        torch.cuda.synchronize()
        want = ref.update(t.tolist(), n.tolist(), parents.tolist(), counts.tolist(), 900, 16, 1)
        got = _lists((up.new_table, up.new_lengths, up.slots, up.granted, up.src, up.dst))
        assert got == [list(w) for w in want], step
        want = ref.compact(t.tolist(), n.tolist(), 900, 16)
        assert _lists((co.new_table, co.src, co.dst, co.used)) == [list(w) for w in want], step
        t.copy_(up.new_table)
        n.copy_(up.new_lengths)
        parents.copy_(_i32([rng.randrange(50) for _ in range(50)], device))
        up.launch()  # an eager launch on the same workspace
        torch.cuda.synchronize()
