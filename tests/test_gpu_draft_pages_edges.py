"""cache_keep and cache_bounds where they could go wrong unseen: the largest tables, keys and values in one tensor."""
from __future__ import annotations

import pytest
import torch

pytestmark = pytest.mark.gpu
BF16 = torch.bfloat16


@pytest.fixture(scope="module")
def ops(pkg, device):
    pkg.torch_ops()
    return torch.ops.mhcpre


def test_bounds_of_the_widest_rows(ops, device):
    """2^30 columns, whose heads take three groups of a workgroup's pieces each: more items of a row than 31 bits count.
    All columns but the first and the last are holes."""
    width, kv_heads, d, pages = 2 ** 30, 24, 256, 9
    table = torch.full((1, width), -1, dtype=torch.int32, device=device)
    table[0, 0], table[0, 2 ** 29 + 5], table[0, 2 ** 30 - 2], table[0, 2 ** 30 - 1] = 3, 5, 7, 1
    k = torch.randn(pages, 1, kv_heads, d, device=device).to(BF16)
    lo, hi = (torch.full((pages, kv_heads, d), 9.0, dtype=BF16, device=device) for _ in range(2))
    length = torch.tensor([width], dtype=torch.int32, device=device)
    ops.cache_bounds(k, table, length, length, lo, hi, width)
    held = [1, 3, 5, 7]
    others = [0, 2, 4, 6, 8]
    for bound in (lo, hi):
        assert torch.equal(bound[held], k[held, 0]) and (bound[others] == 9.0).all()
