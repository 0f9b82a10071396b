"""cache_keep and cache_bounds where they could go wrong unseen: the largest tables, keys and values in one tensor."""
from __future__ import annotations

import pytest
import torch

import draft_ref as ref
from test_gpu_draft_pages import caches

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


@pytest.mark.parametrize("slot_major", [False, True])
@pytest.mark.parametrize("d,dtype", [(64, BF16), (6, torch.float16), (33, torch.float32)])
def test_keep_where_values_are_the_keys(ops, device, d, dtype, slot_major):
    """One tensor as both caches, and a view of it that only has other strides where there is one head: every node
    moves once, in the path's order."""
    for kv_heads in (1, 8):
        (made,), table = caches(device, 3, 4, kv_heads, d, 400, dtype, slot_major, count=1)
        i32 = dict(dtype=torch.int32, device=device)
        paths = [list(range(1, 300)) + [-1], [0] + list(range(2, 300, 2)) + [-1] * 150, list(range(7, 300)) + [-1] * 7]
        args = table, torch.tensor([400, 377, 310], **i32), torch.tensor([300] * 3, **i32), torch.tensor(
            [(p + [-1] * 300)[:300] for p in paths], **i32)
        want, _ = ref.cache_keep(made, made, *(x.cpu() for x in args))
        same = made if kv_heads > 1 else made.as_strided(made.shape, (*made.stride()[:2], 5, 1))
        ops.cache_keep(made, same, *args)
        assert torch.equal(made.cpu(), want)
