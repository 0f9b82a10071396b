"""draft_attention where a window is shorter than what is new, and where whole waves of a block have no rows."""
from __future__ import annotations

import pytest
import torch

from test_gpu_draft_attention import BF16, F16, check, make, ops  # noqa: F401

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("d,S,heads,kv_heads,longest", [(64, 300, 2, 1, 420), (128, 300, 4, 2, 300), (128, 90, 4, 1, 260),
                                                        (64, 600, 2, 2, 700), (80, 200, 2, 1, 330)])
@pytest.mark.parametrize("window", [17, 64, 129, 250])
def test_chains_longer_than_their_window(ops, device, d, S, heads, kv_heads, longest, window):  # noqa: F811
    """Blocks of four and of eight waves of rows, whose first rows see nothing of what the last ones see."""
    a = make(device, 2, S, heads, kv_heads, d, 16, longest, BF16, lengths=[longest, longest - 45], drafted=[S, S - 70],
             tree=False, seed=window)
    check(ops, a, window=window)


@pytest.mark.parametrize("window", [3, 40])
@pytest.mark.parametrize("d,S,heads,kv_heads", [(128, 90, 4, 1), (64, 250, 2, 1)])
def test_trees_deeper_than_their_window(ops, device, d, S, heads, kv_heads, window):  # noqa: F811
    a = make(device, 2, S, heads, kv_heads, d, 16, S + 90, F16, drafted=[S, S - 30])
    depth = torch.arange(-1, S - 1, dtype=torch.int32, device=device).expand(2, S).contiguous()
    a["parents"] = torch.where(torch.arange(S, device=device) % 5 == 4, (depth - 3).clamp(min=-1), depth).int().contiguous()
    check(ops, a, window=window)


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("d,S,heads,kv_heads", [(128, 32, 8, 2), (64, 40, 16, 2), (256, 30, 8, 2), (96, 24, 8, 1)])
def test_rows_that_fill_few_waves(ops, device, dtype, d, S, heads, kv_heads):  # noqa: F811
    """Uneven trees: of some sequences one node, of some none, of some all."""
    drafted = [1, S, 0, 7, S // 2, 9]
    a = make(device, 6, S, heads, kv_heads, d, 16, 300, dtype, lengths=[300, 290, 280, 7, 260, 0], drafted=drafted)
    check(ops, a)
    check(ops, a, window=20)
