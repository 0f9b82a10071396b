"""Sizes at the ends of what the operators for drafted tokens and selected pages take, without a GPU."""
from __future__ import annotations

import pytest

from test_draft_host import keep, lib, sparse  # noqa: F401
from test_serve_host import D, I32, S, call, code


@pytest.mark.parametrize("width,want", [(2 ** 30, "SUCCESS"), (2 ** 30 + 1, "UNSUPPORTED_SHAPE"),
                                        (2 ** 31 - 64, "UNSUPPORTED_SHAPE"), (2 ** 31 - 1, "UNSUPPORTED_SHAPE")])
def test_columns_that_selected_pages_may_have(pkg, lib, width, want):  # noqa: F811
    """A step of the scores or of the selection beyond the last column is an index of 31 bits."""
    over = dict(k=S([20, 1, 2, 64]), v=S([20, 1, 2, 64]), table=D([3, width], I32))
    assert call(pkg, lib, "mhcSparseAttention", sparse(**over))[0] == code(pkg, want)


@pytest.mark.parametrize("nodes,want", [(2 ** 30, "SUCCESS"), (2 ** 30 + 1, "UNSUPPORTED_SHAPE"),
                                        (2 ** 31 - 1, "UNSUPPORTED_SHAPE")])
def test_nodes_that_a_path_may_have(pkg, lib, nodes, want):  # noqa: F811
    """The kernel's steps along a path end behind its last node, in 31 bits."""
    assert call(pkg, lib, "mhcCacheKeep", keep(path=D([3, nodes], I32)))[0] == code(pkg, want)
