"""The executor classes of serve.py take tensors of one GPU only: a host address must not reach a kernel."""
from __future__ import annotations

import pytest
import torch


def _calls(pkg, device):
    i32 = dict(dtype=torch.int32, device=device)
    q, k = torch.zeros(3, 4, 64, dtype=torch.float16, device=device), torch.zeros(3, 2, 64, dtype=torch.float16, device=device)
    cache, positions = torch.zeros(5, 4, 2, 64, dtype=torch.float16, device=device), torch.zeros(3, **i32)
    table, row = torch.zeros(3, 2, **i32), torch.zeros(3, **i32)
    return {
        pkg.QkNormRopeOp: dict(q=q, k=k, positions=positions),
        pkg.PagedAttentionOp: dict(q=q, k_cache=cache, v_cache=cache.clone(), page_table=table, lengths=row),
        pkg.CacheUpdateOp: dict(page_table=table, lengths=row, parents=row, counts=row, pages=5, page_size=4),
        pkg.CacheCompactOp: dict(page_table=table, lengths=row, pages=5, page_size=4),
        pkg.CopyPagesOp: dict(k_cache=cache, v_cache=cache.clone(), src=row, dst=row)}


NAMES = ["QkNormRopeOp", "PagedAttentionOp", "CacheUpdateOp", "CacheCompactOp", "CopyPagesOp"]


@pytest.mark.parametrize("name", NAMES)
def test_host_tensors_are_refused(pkg, name):
    op = getattr(pkg, name)
    with pytest.raises(ValueError, match="one GPU"):
        op(**_calls(pkg, "cpu")[op])


@pytest.mark.gpu
@pytest.mark.parametrize("name", NAMES)
def test_one_host_tensor_is_refused(pkg, device, name):
    """Any one of the tensors on the host, an output or a workspace among them."""
    op = getattr(pkg, name)
    args = _calls(pkg, device)[op]
    op(**args).launch()
    torch.cuda.synchronize()
    for key, value in args.items():
        if isinstance(value, torch.Tensor):
            with pytest.raises(ValueError, match="one GPU"):
                op(**{**args, key: value.cpu()})
    if op is pkg.PagedAttentionOp:
        for key, value in (("out", args["q"].cpu()), ("lse", torch.zeros(3, 4)),
                           ("workspace", torch.empty(1 << 20, dtype=torch.uint8))):
            with pytest.raises(ValueError, match="one GPU"):
                op(**args, **{key: value})
