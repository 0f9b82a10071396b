"""cache_update and cache_compact on the widest table there may be, and nearly full pools."""
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


WIDTH = 2 ** 31 - 1


def _i32(v, device):
    return torch.tensor(v, dtype=torch.int32, device=device)


def test_the_widest_table(ops, device):
    """One row of 2^31 - 1 columns of one token each: holes, and pages at its start and end.  It grows by its last
    column, and is full in the second step."""
    table = torch.full((1, WIDTH), -1, dtype=torch.int32, device=device)
    ends = {0: 9, 1: 3, 1000: 4, WIDTH - 1025: 1, WIDTH - 66: 0, WIDTH - 3: 7}
    for column, page in ends.items():
        table[0, column] = page
    table[0, WIDTH - 1] = 5  # beyond the length: free
    zero, one = _i32([0], device), _i32([1], device)
    new, lengths, slots, granted, src, dst = ops.cache_update(table, _i32([WIDTH - 1], device), zero, one, 10, 1, 1)
    assert lengths.tolist() == [WIDTH] and granted.tolist() == [1] and slots.tolist() == [[2]]
    assert src.tolist() == [-1] and dst.tolist() == [-1]
    table[0, WIDTH - 1] = 2
    assert torch.equal(new, table)
    new.fill_(-7)
    del new
    new, lengths, slots, granted, _, _ = ops.cache_update(table, lengths, zero, one, 10, 1, 1)
    assert lengths.tolist() == [WIDTH] and granted.tolist() == [0] and slots.tolist() == [[-1]]
    assert torch.equal(new, table)
    del new
    # Held: 0, 1, 2, 3, 4, 7, 9; so 7 and 9 move to 5 and 6.
    new, src, dst, used = ops.cache_compact(table, lengths, 10, 1)
    assert src.tolist() == [7, 9, -1, -1, -1] and dst.tolist() == [5, 6, -1, -1, -1] and used.tolist() == [7]
    table[0, 0], table[0, WIDTH - 3] = 6, 5
    assert torch.equal(new, table)


@pytest.mark.parametrize("pages,free", [(40000, 1), (262144, 40), (262144, 1), (300001, 33)])
def test_nearly_full_pools(ops, device, pages, free):
    """The free pages far apart, or all at the pool's start or end: plans as the plain form's."""
    rng = random.Random(pages + free)
    width = 2048
    for where in ("spread", "start", "end"):
        at = set(rng.sample(range(pages), free) if where == "spread" else
                 range(free) if where == "start" else range(pages - free, pages))
        held = [p for p in range(pages) if p not in at]
        rng.shuffle(held)
        table = [held[i:i + width] for i in range(0, len(held), width)]
        lengths = [4 * len(row) for row in table]
        table = [row + [-1] * (width + 8 - len(row)) for row in table]
        t, n = _i32(table, device), _i32(lengths, device)
        got = [o.cpu().tolist() for o in ops.cache_compact(t, n, pages, 4)]
        assert got == [list(w) for w in ref.compact(table, lengths, pages, 4)], where
        rows = list(range(len(table)))
        counts = [1] * len(rows)
        got = [o.cpu().tolist() for o in ops.cache_update(t, n, _i32(rows, device), _i32(counts, device), pages, 4, 1)]
        assert got == [list(w) for w in ref.update(table, lengths, rows, counts, pages, 4, 1)], where
