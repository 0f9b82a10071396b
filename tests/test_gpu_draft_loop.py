"""The operators for drafted tokens and selected pages together: the serving example's loop with trees, and a step of
them under torch.compile and captured into one graph."""
from __future__ import annotations

import sys
from pathlib import Path

import pytest
import torch

import draft_ref as ref

pytestmark = pytest.mark.gpu

sys.path.insert(0, str(Path(__file__).resolve().parents[1] / "examples"))


@pytest.fixture(scope="module")
def ops(pkg, device):
    pkg.torch_ops()
    return torch.ops.mhcpre


@pytest.mark.parametrize("draft,seed", [(1, 0), (5, 1), (12, 2)])
def test_loop_with_drafts(ops, device, draft, seed):
    """Every row's last confirmed token, through trees, kept paths, forks and compactions, against the attention without
    a cache.  Values are below 4: the output's rounding to bf16 is off by up to 2^-9 * 4 = 0.008, and q, k and v by a
    last bit (2^-8 of themselves, 0.016 of a value) where sums of batches of another shape round the other way, which
    moves scores of size 1 by 2 * 2^-8 and so the mean of values by up to 2 * 2^-8 * 4 = 0.03: 0.05 at most."""
    import serve_block

    said = []
    worst = serve_block.serve(steps=20, check=True, seed=seed, say=said.append, draft=draft)
    assert worst < 0.05, said
    assert any("compaction" in line for line in said)


def _state(device):
    g = torch.Generator(device=device).manual_seed(0)
    rand = lambda *s: torch.randn(*s, generator=g, device=device).to(torch.bfloat16)  # noqa: E731
    i32 = lambda v: torch.tensor(v, dtype=torch.int32, device=device)  # noqa: E731
    return dict(q=rand(3, 6, 4, 64), one=rand(3, 4, 64), k=rand(20, 16, 2, 64), v=rand(20, 16, 2, 64),
                lo=-rand(20, 2, 64).abs(), hi=rand(20, 2, 64).abs(), table=i32([[0, 2, 9], [3, 1, 8], [11, 4, 5]]),
                lengths=i32([17, 40, 6]), drafted=i32([6, 5, 6]),
                parents=i32([[-1, 0, 0, 1, 2, 4], [-1, 0, 1, 2, 3, 4], [-1, 0, 0, 0, 1, 1]]),
                tokens=torch.tensor([[0, 1, 2, 2, 1, 0], [0, 1, 1, 2, 0, 0], [3, 1, 2, 0, 2, 1]], device=device),
                chosen=torch.tensor([[2, 0, 1, 0, 0, 5], [1, 1, 2, 7, 0, 0], [0, 0, 0, 9, 0, 0]], device=device))


def _step(ops, a):
    out, lse = ops.draft_attention(a["q"], a["k"], a["v"], a["table"], a["lengths"], a["drafted"], a["parents"])
    path, accepted, nxt, lengths = ops.draft_accept(a["tokens"], a["parents"], a["drafted"], a["chosen"], a["lengths"])
    ops.cache_keep(a["k"], a["v"], a["table"], a["lengths"], a["drafted"], path)
    ops.cache_bounds(a["k"], a["table"], lengths, accepted, a["lo"], a["hi"], 6)
    some, some_lse, columns = ops.sparse_attention(a["one"], a["k"], a["v"], a["lo"], a["hi"], a["table"], lengths, 2)
    return out.float() * 2, lse, path, accepted, nxt, lengths, some, some_lse, columns


def test_a_step_against_the_plain_forms(ops, device):
    a, b = _state(device), _state(device)
    out, lse, path, accepted, nxt, lengths, some, _, columns = _step(ops, a)
    want, _, bound, _ = ref.draft_attention(b["q"], b["k"], b["v"], b["table"], b["lengths"], b["drafted"], b["parents"],
                                            64 ** -0.5)
    assert ((out.cpu().double() / 2 - want).abs() <= bound).all()
    lists = [b[k].tolist() for k in ("tokens", "parents", "drafted", "chosen", "lengths")]
    assert [t.tolist() for t in (path, accepted, nxt, lengths)] == list(ref.draft_accept(*lists))
    k, v = ref.cache_keep(b["k"], b["v"], b["table"].cpu(), b["lengths"].cpu(), b["drafted"].cpu(), path.cpu())
    assert torch.equal(a["k"].cpu(), k) and torch.equal(a["v"].cpu(), v)
    lo, hi = ref.cache_bounds(k, b["table"].cpu(), lengths.cpu(), accepted.cpu(), b["lo"], b["hi"], 6)
    assert torch.equal(a["lo"].cpu().double(), lo) and torch.equal(a["hi"].cpu().double(), hi)
    want, _, bound, _, want_columns = ref.sparse_attention(b["one"], k, v, lo, hi, b["table"], lengths.cpu(), 2, 1, 1,
                                                           64 ** -0.5)
    assert torch.equal(columns.cpu(), want_columns)
    assert ((some.cpu().double() - want).abs() <= bound).all()


def test_a_step_under_torch_compile(ops, device):
    a, b = _state(device), _state(device)
    want = _step(ops, a)
    got = torch.compile(lambda b: _step(ops, b), backend="aot_eager", fullgraph=True)(b)
    assert all(torch.equal(x, y) for x, y in zip(got, want))
    assert all(torch.equal(a[k], b[k]) for k in ("k", "v", "lo", "hi"))
    assert not torch.equal(a["k"], _state(device)["k"])


@pytest.mark.parametrize("name,keys", [
    ("draft_attention", "q k v table lengths drafted parents"), ("draft_accept", "tokens parents drafted chosen lengths"),
    ("cache_keep", "k v table lengths drafted parents"), ("cache_bounds", "k table lengths drafted lo hi 6"),
    ("sparse_attention", "one k v lo hi table lengths 2")])
def test_schemas_and_shapes(ops, device, name, keys):
    a = _state(device)
    torch.library.opcheck(getattr(ops, name).default, tuple(int(k) if k.isdigit() else a[k] for k in keys.split()))


def test_a_step_in_a_graph(ops, device):
    """All of them captured together, with the allocator's own memory; replayed on other contents."""
    a = _state(device)
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        _step(ops, a)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = _step(ops, a)
    g = torch.Generator(device=device).manual_seed(5)
    for n in (40, 6, 21, 33):
        fresh = _state(device)
        fresh["lengths"].fill_(n)
        fresh["chosen"].copy_(torch.randint(0, 3, (3, 6), generator=g, device=device))
        fresh["q"].copy_(torch.randn(fresh["q"].shape, generator=g, device=device))
        for key in a:
            a[key].copy_(fresh[key])
        want = _step(ops, fresh)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(x, y) for x, y in zip(got, want))
        assert all(torch.equal(a[k], fresh[k]) for k in ("k", "v", "lo", "hi"))
