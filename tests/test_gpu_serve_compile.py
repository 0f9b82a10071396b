"""The serving operators under torch.compile, those that change their arguments among them, and torch's own checks
of their schemas and shape functions."""
from __future__ import annotations

import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ops(pkg, device):
    pkg.torch_ops()
    return torch.ops.mhcpre


def _args(device):
    g = torch.Generator(device=device).manual_seed(0)
    rand = lambda *s: torch.randn(*s, generator=g, device=device).to(torch.bfloat16)  # noqa: E731
    i32 = lambda v: torch.tensor(v, dtype=torch.int32, device=device)  # noqa: E731
    return dict(q=rand(3, 4, 64), k=rand(3, 2, 64), v=rand(3, 2, 64), positions=torch.arange(3, device=device),
                inv_freq=10000.0 ** (-torch.arange(0, 64, 2, dtype=torch.float64, device=device) / 64),
                k_cache=rand(6, 16, 2, 64), v_cache=rand(6, 16, 2, 64), table=i32([[0, 2], [3, 1], [1, 4]]),
                lengths=i32([17, 30, 3]), parents=i32([0, 0, -1]), counts=i32([1, 1, 1]))


def _step(ops, a):
    table, lengths, slots, granted, src, dst = ops.cache_update(a["table"], a["lengths"], a["parents"], a["counts"], 6, 16)
    ops.cache_copy_pages(a["k_cache"], a["v_cache"], src, dst)
    q = ops.qk_norm_rope_append(a["q"], a["k"], a["v"], a["positions"], a["inv_freq"], slots.view(-1), a["k_cache"],
                                a["v_cache"])
    out, lse = ops.paged_attention(q, a["k_cache"], a["v_cache"], table, lengths)
    table, src, dst, used = ops.cache_compact(table, lengths, 6, 16)
    ops.cache_copy_pages(a["k_cache"], a["v_cache"], src, dst)
    return out.float() * 2, lse, table, lengths, granted, used


def test_a_step_under_torch_compile(ops, device):
    a, b = _args(device), _args(device)
    want = _step(ops, a)
    got = torch.compile(lambda b: _step(ops, b), backend="aot_eager", fullgraph=True)(b)
    assert all(torch.equal(x, y) for x, y in zip(got, want))
    assert torch.equal(a["k_cache"], b["k_cache"]) and torch.equal(a["v_cache"], b["v_cache"])
    assert not torch.equal(a["k_cache"], _args(device)["k_cache"])


@pytest.mark.parametrize("name,keys", [
    ("qk_norm_rope", "q k positions inv_freq"), ("qk_norm_rope_append", "q k v positions inv_freq slots k_cache v_cache"),
    ("paged_attention", "q k_cache v_cache table lengths"), ("cache_update", "table lengths parents counts 6 16 2"),
    ("cache_compact", "table lengths 6 16"), ("cache_copy_pages", "k_cache v_cache src dst")])
def test_schemas_and_shapes(ops, device, name, keys):
    a = _args(device)
    a.update(slots=torch.tensor([1, 17, -1], device=device), src=a["counts"][:2] - 2, dst=a["counts"][:2] + 2)
    torch.library.opcheck(getattr(ops, name).default, tuple(int(k) if k.isdigit() else a[k] for k in keys.split()))
