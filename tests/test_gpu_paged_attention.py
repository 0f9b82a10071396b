"""paged_attention against a plain 64-bit implementation."""
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


def _state(device, B, heads, kv_heads, d, page, lengths, dtype, seed=0, width=None, extra=3, slot_major=False, q_scale=2.0):
    g = torch.Generator().manual_seed(seed)
    need = [-(-n // page) for n in lengths]
    pages = sum(need) + extra
    width = max(max(need), 1) if width is None else width
    perm = torch.randperm(pages, generator=g).int()
    table = torch.full((B, width), -1, dtype=torch.int32)
    at = 0
    for b, n in enumerate(need):
        n = min(n, width)
        table[b, :n] = perm[at:at + n]
        at += n
    shape = (pages, page, kv_heads, d) if slot_major else (pages, kv_heads, page, d)
    caches = []
    for _ in range(2):
        c = torch.randn(shape, generator=g).to(dtype).to(device)
        caches.append(c if slot_major else c.transpose(1, 2))
    q = (q_scale * torch.randn(B, heads, d, generator=g)).to(dtype).to(device)
    return q, caches[0], caches[1], table.to(device), torch.tensor(lengths, dtype=torch.int32, device=device)


def _check(out, lse, want):
    w_out, w_lse, b_out, b_lse = want
    out, lse = out.cpu().double(), lse.cpu().double()
    empty = torch.isinf(w_lse)
    assert torch.equal(torch.isinf(lse) & (lse < 0), empty)
    off = (out - w_out).abs()
    assert (off <= b_out).all(), f"out: {(off / b_out).max():.3g} of its bound"
    off = (lse - w_lse)[~empty].abs()
    assert (off <= b_lse[~empty]).all(), f"lse: {(off / b_lse[~empty]).max():.3g} of its bound"


def _run(ops, state, scale=None, window=0):
    q = state[0]
    scale = q.shape[-1] ** -0.5 if scale is None else scale
    out, lse = ops.paged_attention(*state, scale, window)
    assert out.dtype == q.dtype and out.shape == q.shape and lse.shape == q.shape[:-1]
    _check(out, lse, ref.attention(*state, scale, window))
    return out, lse


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("d", [32, 64, 80, 96, 112, 128, 160, 192, 256])
def test_head_sizes(ops, device, d, dtype):
    _run(ops, _state(device, 3, 8, 2, d, 16, [1, 77, 300], dtype, seed=d))


@pytest.mark.parametrize("heads,kv_heads", [(1, 1), (5, 5), (3, 1), (7, 1), (16, 1), (17, 1), (40, 2), (64, 1), (65, 1),
                                            (130, 1), (12, 4)])
def test_head_groups(ops, device, heads, kv_heads):
    _run(ops, _state(device, 2, heads, kv_heads, 64, 8, [33, 150], torch.bfloat16, seed=heads))


@pytest.mark.parametrize("page", [1, 3, 7, 16, 64, 100, 256])
def test_page_sizes_and_lengths(ops, device, page):
    """Lengths about every tile and page edge, in one ragged batch, of any order."""
    lengths = [0, 1, 2, 15, 16, 17, 31, 32, 33, 63, 64, 65, 127, 128, 129, 255, 257, 511, 513, 1025, page, page + 1,
               max(page - 1, 0), 0]
    _run(ops, _state(device, len(lengths), 4, 2, 64, page, lengths, torch.float16, seed=page))


@pytest.mark.parametrize("window", [1, 2, 31, 32, 33, 100, 128, 129, 5000])
def test_windows(ops, device, window):
    _run(ops, _state(device, 5, 4, 1, 64, 16, [0, 1, 33, 400, 777], torch.bfloat16, seed=window), window=window)


@pytest.mark.parametrize("slot_major", [False, True])
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_long_few_rows(ops, device, dtype, slot_major):
    """One and two long rows: their length is split over many workgroups and joined."""
    _run(ops, _state(device, 1, 8, 1, 128, 64, [20011], dtype, slot_major=slot_major))
    _run(ops, _state(device, 2, 4, 2, 128, 16, [9000, 3], dtype, seed=1, slot_major=slot_major))


@pytest.mark.parametrize("heads,kv_heads,d,lengths,window", [
    (1, 1, 32, [66000], 0), (16, 1, 64, [70000], 0), (40, 1, 192, [33000], 0), (24, 4, 128, [20000], 0),
    (32, 2, 256, [10000, 7001], 0), (17, 1, 80, [40000, 5], 30000), (12, 1, 112, [300, 24000, 0, 26000], 0)])
def test_rows_of_many_parts(pkg, ops, device, heads, kv_heads, d, lengths, window):
    """So many workgroups at a row that their parts are joined in spans first; again on a workspace that holds anything."""
    state = _state(device, len(lengths), heads, kv_heads, d, 64, lengths, torch.bfloat16, seed=d)
    out, lse = _run(ops, state, window=window)
    op = pkg.PagedAttentionOp(*state, window=window)
    for fill in (0, 255, 7):
        op.workspace.fill_(fill)
        for _ in range(2):
            op.out.fill_(3.0)
            op.launch()
            assert torch.equal(op.out, out) and torch.equal(op.lse, lse)


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("B,heads,kv_heads,d,page,most,window", [
    (300, 8, 8, 32, 16, 90, 0), (1100, 3, 1, 64, 7, 40, 0), (150, 16, 8, 128, 64, 300, 0), (260, 20, 4, 80, 1, 65, 0),
    (280, 4, 2, 256, 16, 48, 0), (270, 4, 4, 96, 16, 3000, 37), (2100, 1, 1, 112, 32, 33, 1)])
def test_many_short_rows(ops, device, B, heads, kv_heads, d, page, most, window, dtype):
    """Large batches of rows that the table's width or the window keeps short: empty ones and holes among them."""
    lengths = [(i * i * 37) % (most + 1) for i in range(B)]
    state = _state(device, B, heads, kv_heads, d, page, lengths, dtype, seed=B)
    state[3][::11, 0] = -1
    _run(ops, state, window=window)


def test_large_ragged_batch(ops, device):
    lengths = [(i * i * 37) % 701 for i in range(300)]
    _run(ops, _state(device, 300, 6, 2, 32, 16, lengths, torch.float16))


def test_no_key_and_no_row(ops, device):
    state = _state(device, 3, 4, 2, 64, 16, [0, 0, 0], torch.float16)
    out, lse = ops.paged_attention(*state)
    assert (out == 0).all() and torch.isneginf(lse).all()
    q, k, v, table, lengths = state
    out, lse = ops.paged_attention(q[:0], k, v, table[:0], lengths[:0])
    assert out.shape == (0, 4, 64) and lse.shape == (0, 4)


def test_holes_and_lengths_out_of_range(ops, device):
    q, k, v, table, lengths = _state(device, 4, 4, 2, 64, 8, [200, 64, 64, 100], torch.bfloat16)
    table[0, 3] = -1
    table[0, 7] = k.shape[0]  # one beyond the pool
    table[0, 8] = 2 ** 31 - 1
    table[1, :] = -5  # a row of holes only
    lengths[2] = -7
    lengths[3] = 10 ** 9  # beyond the table's width: all of it, -1 entries included
    out, lse = _run(ops, (q, k, v, table, lengths))
    assert (out[1:3] == 0).all() and torch.isneginf(lse[1:3]).all()


@pytest.mark.parametrize("bad", [math.nan, math.inf, -math.inf])
def test_unseen_slots_may_hold_anything(ops, device, bad):
    """Slots beyond a row's length, before its window and of pages of nobody's are not read into results."""
    for window in (0, 50):
        q, k, v, table, lengths = _state(device, 3, 4, 2, 64, 16, [5, 100, 131], torch.float16)
        seen = torch.zeros(k.shape[:2], dtype=torch.bool)
        for b, n in enumerate(lengths.tolist()):
            for t in range(max(0, n - window) if window else 0, n):
                seen[int(table[b, t // 16]), t % 16] = True
        want = ref.attention(q, k, v, table, lengths, 0.125, window)
        k[~seen.to(device)] = bad
        v[~seen.to(device)] = bad
        _check(*ops.paged_attention(q, k, v, table, lengths, 0.125, window), want)


def test_extreme_scores(ops, device):
    """Scores far apart (one key has all the weight), equal, and of the type's largest keys."""
    state = _state(device, 2, 4, 2, 64, 16, [77, 513], torch.bfloat16, q_scale=100.0)
    _run(ops, state, scale=1.0)
    _run(ops, state, scale=0.0)
    _run(ops, state, scale=-0.125)
    q, k, v, table, lengths = state
    k = (k.float() * 2.0 ** 100).to(torch.bfloat16)
    _run(ops, ((q.float() * 2.0 ** -100).to(torch.bfloat16), k, v, table, lengths), scale=0.01)


def test_subnormal_and_tiny_weights(ops, device):
    """A long row whose weights are each far below the type's smallest normal value sums up right."""
    state = _state(device, 1, 2, 1, 64, 64, [70000], torch.float16, q_scale=0.05)
    _run(ops, state)


def test_infinite_key_gives_its_value(ops, device):
    """A key at -inf in a direction that the query has positive is never seen (its weight is 0)."""
    q, k, v, table, lengths = _state(device, 1, 2, 1, 64, 16, [40], torch.float16)
    q.abs_()
    k[int(table[0, 1]), 3, 0, 7] = -math.inf
    out, lse = ops.paged_attention(q, k, v, table, lengths)
    k2 = k.clone()
    table2 = table.clone()
    keep = [t for t in range(40) if t != 19]
    kk = torch.stack([k2[int(table[0, t // 16]), t % 16] for t in keep])
    vv = torch.stack([v[int(table[0, t // 16]), t % 16] for t in keep])
    table2 = torch.arange(39, dtype=torch.int32, device=device).view(1, 39)
    want = ref.attention(q, kk[:, None], vv[:, None], table2, torch.tensor([39]), 0.125)
    _check(out, lse, want)


def test_rows_do_not_depend_on_the_batch(ops, device):
    """A row alone and the same row in a batch give the same bits where the split is the same, and results within
    the bounds anyway; a call repeated gives the same bits."""
    state = _state(device, 7, 8, 2, 128, 16, [1000, 3, 0, 512, 700, 65, 999], torch.bfloat16)
    a = _run(ops, state)
    for _ in range(5):
        b = ops.paged_attention(*state)
        assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])
    q, k, v, table, lengths = state
    for b in range(7):
        _run(ops, (q[b:b + 1], k, v, table[b:b + 1], lengths[b:b + 1]))


def test_strides_and_leading_dimensions(ops, device):
    q, k, v, table, lengths = _state(device, 4, 6, 2, 64, 16, [50, 3, 200, 17], torch.float16)
    want = ops.paged_attention(q, k, v, table, lengths)
    wide = torch.zeros(4, 1, 9, 64, dtype=q.dtype, device=device)
    wide[:, 0, 2:8] = q
    got = ops.paged_attention(wide[:, :, 2:8], k, v, table, lengths)
    assert got[0].shape == (4, 1, 6, 64) and got[1].shape == (4, 1, 6)
    assert torch.equal(got[0][:, 0], want[0]) and torch.equal(got[1][:, 0], want[1])
    odd = torch.zeros(4 * 6 * 64 + 3, dtype=q.dtype, device=device)[3:].view(4, 6, 64)  # not 16-byte aligned
    odd.copy_(q)
    assert torch.equal(ops.paged_attention(odd, k, v, table, lengths)[0], want[0])
    # Pages, slots and heads in other orders and with gaps.
    for order in ((0, 1, 2), (1, 0, 2), (2, 1, 0), (0, 2, 1), (2, 0, 1)):
        dims = [k.shape[i] for i in order]
        caches = []
        for c in (k, v):
            big = torch.full([dims[0], dims[1] + 1, dims[2], 72], math.nan, dtype=k.dtype, device=device)
            view = big[:, :dims[1], :, :64].permute(*[order.index(i) for i in range(3)], 3)
            view.copy_(c)
            caches.append(view)
        got = ops.paged_attention(q, *caches, table, lengths)
        assert torch.equal(got[0], want[0]), order


def test_cache_beyond_32_bits(ops, device):
    """Pages whose elements lie beyond 2^32 bytes and 2^32 elements of the cache's start."""
    pages, page, kv_heads, d = 70000, 64, 8, 128  # 4.6e9 elements each
    k = torch.empty(pages, kv_heads, page, d, dtype=torch.bfloat16, device=device).transpose(1, 2)
    v = torch.empty(pages, kv_heads, page, d, dtype=torch.bfloat16, device=device).transpose(1, 2)
    use = [69999, 0, 32768, 65536, 40000]
    for c in (k, v):
        for p in use:
            c[p] = torch.randn(page, kv_heads, d, device=device)
    q = torch.randn(1, 16, d, device=device).to(torch.bfloat16)
    table = torch.tensor([use], dtype=torch.int32, device=device)
    lengths = torch.tensor([5 * page - 3], dtype=torch.int32, device=device)
    out, lse = ops.paged_attention(q, k, v, table, lengths)
    small = torch.arange(5, dtype=torch.int32).view(1, 5)
    _check(out, lse, ref.attention(q, k[use], v[use], small, lengths, d ** -0.5))


def test_on_another_stream_and_executor(pkg, ops, device):
    state = _state(device, 3, 8, 2, 128, 16, [40, 3000, 1], torch.bfloat16)
    want = ops.paged_attention(*state)
    op = pkg.PagedAttentionOp(*state)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    op.workspace.fill_(255)  # any contents
    side.wait_stream(torch.cuda.current_stream())
    for _ in range(3):
        op.launch(side)
    side.synchronize()
    assert torch.equal(op.out, want[0]) and torch.equal(op.lse, want[1])
    no_lse = pkg.PagedAttentionOp(*state, lse=False)
    no_lse.launch()
    torch.cuda.synchronize()
    assert no_lse.lse is None and torch.equal(no_lse.out, want[0])


def test_graph_replays(pkg, ops, device):
    """Replays see the tensors' contents of their own time; eager launches on the same workspace in between."""
    q, k, v, table, lengths = _state(device, 3, 8, 2, 64, 16, [900, 3000, 1], torch.float16)
    op = pkg.PagedAttentionOp(q, k, v, table, lengths)
    op.launch()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        op.launch()
    for step, n in enumerate(([900, 3000, 1], [10, 0, 1], [900, 2999, 16], [0, 0, 0], [1, 3000, 15])):
        lengths.copy_(torch.tensor(n, dtype=torch.int32))
        q.normal_()
        op.out.fill_(7)
        graph.replay()
        torch.cuda.synchronize()
        want = ops.paged_attention(q, k, v, table, lengths)
        assert torch.equal(op.out, want[0]) and torch.equal(op.lse, want[1]), step
        op.launch()
        torch.cuda.synchronize()
        assert torch.equal(op.out, want[0])
