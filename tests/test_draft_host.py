"""The host side of the operators for drafted tokens and selected pages, without a GPU: refusals, workspaces, shapes for
tracing, and the plain implementations that the GPU tests compare with."""
from __future__ import annotations

import math

import pytest
import torch
from torch._subclasses.fake_tensor import FakeTensorMode

import draft_ref as ref
from test_serve_host import BF16, BIG, D, F16, F32, F64, FAKE, I32, I64, S, call, code


@pytest.fixture(scope="module")
def lib(pkg):
    return pkg.load_serve_library()


def draft(**over):
    a = dict(q=S([3, 5, 8, 64]), k=S([20, 16, 2, 64]), v=S([20, 16, 2, 64]), table=D([3, 5], I32), lengths=D([3], I32),
             drafted=D([3], I32), parents=D([3, 5], I32), scale=0.125, window=0, out=S([3, 5, 8, 64]),
             lse=D([3, 5, 8], F32))
    assert set(over) <= set(a)
    return list({**a, **over}.values())


def accept(**over):
    a = dict(tokens=D([3, 5], I64), parents=D([3, 5], I32), drafted=D([3], I32), chosen=D([3, 5], I64),
             lengths=D([3], I32), path=D([3, 5], I32), accepted=D([3], I32), next=D([3], I64), new_lengths=D([3], I32))
    assert set(over) <= set(a)
    return list({**a, **over}.values())


def keep(**over):
    a = dict(k=S([20, 16, 2, 64]), v=S([20, 16, 2, 64]), table=D([3, 5], I32), lengths=D([3], I32), drafted=D([3], I32),
             path=D([3, 9], I32))
    assert set(over) <= set(a)
    return list({**a, **over}.values())


def bounds(**over):
    a = dict(k=S([20, 16, 2, 64]), table=D([3, 5], I32), lengths=D([3], I32), counts=D([3], I32), tokens=7,
             lo=S([20, 2, 64]), hi=S([20, 2, 64]))
    assert set(over) <= set(a)
    return list({**a, **over}.values())


def sparse(**over):
    a = dict(q=S([3, 8, 64]), k=S([20, 16, 2, 64]), v=S([20, 16, 2, 64]), lo=S([20, 2, 64]), hi=S([20, 2, 64]),
             table=D([3, 5], I32), lengths=D([3], I32), top=4, first=1, last=2, scale=0.125, out=S([3, 8, 64]),
             lse=D([3, 8], F32), columns=D([3, 2, 4], I32))
    assert set(over) <= set(a)
    return list({**a, **over}.values())


OPS = {"mhcDraftAttention": draft, "mhcDraftAccept": accept, "mhcCacheKeep": keep, "mhcCacheBounds": bounds,
       "mhcSparseAttention": sparse}


@pytest.mark.parametrize("name", OPS)
def test_valid_calls_and_workspaces(pkg, lib, name):
    assert {name, name + "GetWorkspaceSize"} <= set(pkg.exported_symbols(pkg.serve.SERVE_HEADER))
    st, ws, second = call(pkg, lib, name, OPS[name]())
    assert st == 0
    assert (ws > 0) == (name in ("mhcDraftAttention", "mhcSparseAttention"))
    if ws:
        assert second == [code(pkg, "WORKSPACE_TOO_SMALL")] * 3
    assert getattr(lib, name)(None, 0, None, None) == code(pkg, "NULL_ARGUMENT")


NULLS = [(n, k) for n, f in (("mhcDraftAttention", ("q", "k", "v", "table", "lengths", "drafted", "out")),
                             ("mhcDraftAccept", ("tokens", "drafted", "chosen", "lengths", "path", "accepted", "next",
                                                 "new_lengths")),
                             ("mhcCacheKeep", ("k", "v", "table", "lengths", "drafted", "path")),
                             ("mhcCacheBounds", ("k", "table", "lengths", "counts", "lo", "hi")),
                             ("mhcSparseAttention", ("q", "k", "v", "lo", "hi", "table", "lengths", "out", "columns")))
         for k in f]


@pytest.mark.parametrize("name,key", NULLS)
def test_null_arguments(pkg, lib, name, key):
    assert call(pkg, lib, name, OPS[name](**{key: None}))[0] == code(pkg, "NULL_ARGUMENT")


@pytest.mark.parametrize("over,want", [
    (dict(q=S([3, 8, 64])), "INVALID_SHAPE"), (dict(q=S([3, 5, 7, 64]), out=S([3, 5, 7, 64]), lse=None), "INVALID_SHAPE"),
    (dict(q=S([3, 5, 8, 96])), "INVALID_SHAPE"), (dict(out=S([3, 4, 8, 64])), "INVALID_SHAPE"),
    (dict(q=S([3, 5, 8, 64], F32)), "INVALID_DTYPE"), (dict(q=S([3, 5, 8, 64], F16)), "INVALID_DTYPE"),
    (dict(v=S([20, 16, 2, 64], F16)), "INVALID_DTYPE"), (dict(v=S([19, 16, 2, 64])), "INVALID_SHAPE"),
    (dict(table=D([4, 5], I32)), "INVALID_SHAPE"), (dict(table=D([3, 5], I64)), "INVALID_DTYPE"),
    (dict(drafted=D([2], I32)), "INVALID_SHAPE"), (dict(drafted=D([3], I64)), "INVALID_DTYPE"),
    (dict(parents=D([3, 4], I32)), "INVALID_SHAPE"), (dict(parents=D([3, 5], I64)), "INVALID_DTYPE"),
    (dict(parents=D([3, 5], I32, FAKE + 2)), "MISALIGNED"), (dict(parents=None), "SUCCESS"),
    (dict(window=-1), "INVALID_SHAPE"), (dict(lse=None), "SUCCESS"), (dict(lse=D([3, 5], F32)), "INVALID_SHAPE"),
    (dict(q=S([3, 257, 8, 64]), out=S([3, 257, 8, 64]), parents=D([3, 257], I32), lse=None), "UNSUPPORTED_SHAPE"),
    (dict(q=S([3, 257, 8, 64]), out=S([3, 257, 8, 64]), parents=None, lse=None), "SUCCESS"),
    (dict(q=S([3, 256, 8, 64]), out=S([3, 256, 8, 64]), parents=D([3, 256], I32), lse=None), "SUCCESS"),
    (dict(q=S([3, 2 ** 21, 8, 64]), out=S([3, 2 ** 21, 8, 64]), parents=None, lse=None), "UNSUPPORTED_SHAPE"),
    (dict(q=S([3, 2 ** 20, 8, 64]), out=S([3, 2 ** 20, 8, 64]), parents=None, lse=None, table=D([3, 2 ** 16], I32)),
     "UNSUPPORTED_SHAPE"),
    (dict(q=S([3, 5, 8, 72]), k=S([20, 16, 2, 72]), v=S([20, 16, 2, 72]), out=S([3, 5, 8, 72])), "UNSUPPORTED_SHAPE"),
    (dict(q=S([3, 5, 8, 64], data=FAKE + 8)), "MISALIGNED"),
    (dict(q=S([3, 5, 8, 64], st=[2564, 512, 64, 1])), "MISALIGNED"),
    (dict(q=S([3, 5, 8, 64], st=[99 * 64, 8 * 64, 128, 1])), "SUCCESS"),
    (dict(k=S([BIG, 16, 2, 64]), v=S([BIG, 16, 2, 64])), "UNSUPPORTED_SHAPE"),
    (dict(q=S([3, 0, 8, 64], data=0), out=S([3, 0, 8, 64], data=0), parents=None, lse=None), "SUCCESS"),
    (dict(q=S([0, 5, 8, 64], data=0), table=D([0, 5], I32, 0), lengths=D([0], I32, 0), drafted=D([0], I32, 0),
          parents=D([0, 5], I32, 0), out=S([0, 5, 8, 64], data=0), lse=D([0, 5, 8], F32, 0)), "SUCCESS")])
def test_draft_attention_arguments(pkg, lib, over, want):
    assert call(pkg, lib, "mhcDraftAttention", draft(**over))[0] == code(pkg, want)


@pytest.mark.parametrize("over,want", [
    (dict(tokens=D([3, 5], I32)), "INVALID_DTYPE"),
    (dict(tokens=D([3, 5], I32), chosen=D([3, 5], I32), next=D([3], I32)), "SUCCESS"),
    (dict(tokens=D([3, 5], F32), chosen=D([3, 5], F32), next=D([3], F32)), "INVALID_DTYPE"),
    (dict(parents=None), "SUCCESS"), (dict(tokens=D([3], I64)), "INVALID_SHAPE"),
    (dict(chosen=D([3, 6], I64)), "INVALID_SHAPE"), (dict(next=D([3], I32)), "INVALID_DTYPE"),
    (dict(path=D([3, 5], I64)), "INVALID_DTYPE"), (dict(accepted=D([4], I32)), "INVALID_SHAPE"),
    (dict(lengths=D([3], I32, FAKE + 1)), "MISALIGNED"),
    (dict(tokens=D([3, 257], I64), chosen=D([3, 257], I64), path=D([3, 257], I32), parents=None), "UNSUPPORTED_SHAPE")])
def test_draft_accept_arguments(pkg, lib, over, want):
    assert call(pkg, lib, "mhcDraftAccept", accept(**over))[0] == code(pkg, want)


@pytest.mark.parametrize("over,want", [
    (dict(k=S([20, 16, 2, 64], F32), v=S([20, 16, 2, 64], F32)), "SUCCESS"),
    (dict(k=S([20, 16, 2, 64], I32), v=S([20, 16, 2, 64], I32)), "INVALID_DTYPE"),
    (dict(v=S([20, 16, 2, 32])), "INVALID_SHAPE"), (dict(path=D([4, 9], I32)), "INVALID_SHAPE"),
    (dict(path=D([3], I32)), "INVALID_SHAPE"), (dict(path=D([3, 0], I32, 0)), "SUCCESS"),
    (dict(drafted=D([3], I64)), "INVALID_DTYPE"), (dict(table=D([3, 2 ** 28], I32)), "UNSUPPORTED_SHAPE"),
    (dict(k=S([20, 16, 2, 64], data=FAKE + 1)), "MISALIGNED"), (dict(k=S([20, 16, 2, 64], data=FAKE + 2)), "SUCCESS")])
def test_cache_keep_arguments(pkg, lib, over, want):
    assert call(pkg, lib, "mhcCacheKeep", keep(**over))[0] == code(pkg, want)


@pytest.mark.parametrize("over,want", [
    (dict(k=S([20, 16, 2, 64], F32)), "INVALID_DTYPE"), (dict(lo=S([20, 2, 64], F16)), "INVALID_DTYPE"),
    (dict(hi=S([19, 2, 64])), "INVALID_SHAPE"), (dict(hi=S([20, 1, 2, 64])), "INVALID_SHAPE"),
    (dict(tokens=-1), "INVALID_SHAPE"), (dict(tokens=0), "SUCCESS"), (dict(tokens=2 ** 40), "SUCCESS"),
    (dict(lo=S([20, 2, 64], data=FAKE + 8)), "MISALIGNED"), (dict(counts=D([2], I32)), "INVALID_SHAPE"),
    (dict(k=S([20, 16, 2, 40]), lo=S([20, 2, 40]), hi=S([20, 2, 40])), "UNSUPPORTED_SHAPE")])
def test_cache_bounds_arguments(pkg, lib, over, want):
    assert call(pkg, lib, "mhcCacheBounds", bounds(**over))[0] == code(pkg, want)


@pytest.mark.parametrize("over,want", [
    (dict(top=0, first=0, last=0, columns=D([3, 2, 0], I32, 0)), "INVALID_SHAPE"), (dict(first=-1), "INVALID_SHAPE"),
    (dict(first=3), "INVALID_SHAPE"), (dict(last=4), "INVALID_SHAPE"), (dict(first=2 ** 62, last=2 ** 62), "INVALID_SHAPE"),
    (dict(first=0, last=0), "SUCCESS"), (dict(columns=D([3, 2, 5], I32)), "INVALID_SHAPE"),
    (dict(columns=D([3, 2, 4], I64)), "INVALID_DTYPE"), (dict(lo=S([20, 2, 64], F16)), "INVALID_DTYPE"),
    (dict(hi=S([20, 3, 64])), "INVALID_SHAPE"), (dict(lo=S([20, 2, 64], st=[129, 64, 1])), "MISALIGNED"),
    (dict(top=2 ** 28, columns=D([3, 2, 2 ** 28], I32)), "UNSUPPORTED_SHAPE"), (dict(lse=None), "SUCCESS"),
    (dict(q=S([3, 7, 64]), out=S([3, 7, 64]), lse=None), "INVALID_SHAPE"),
    (dict(q=S([0, 8, 64], data=0), table=D([0, 5], I32, 0), lengths=D([0], I32, 0), out=S([0, 8, 64], data=0),
          lse=D([0, 8], F32, 0), columns=D([0, 2, 4], I32, 0)), "SUCCESS")])
def test_sparse_attention_arguments(pkg, lib, over, want):
    assert call(pkg, lib, "mhcSparseAttention", sparse(**over))[0] == code(pkg, want)


# ---- tracing and host tensors ----------------------------------------------------


def test_shapes_for_tracing(pkg):
    pkg.torch_ops()
    ops = torch.ops.mhcpre
    with FakeTensorMode():
        q, cache = torch.empty(3, 5, 4, 64, dtype=torch.float16), torch.empty(9, 4, 2, 64, dtype=torch.float16)
        bound, table = torch.empty(9, 2, 64, dtype=torch.float16), torch.empty(3, 6, dtype=torch.int32)
        n, nodes = torch.empty(3, dtype=torch.int32), torch.empty(3, 5, dtype=torch.int32)
        out, lse = ops.draft_attention(q, cache, cache, table, n, n, nodes)
        assert out.shape == q.shape and lse.shape == (3, 5, 4) and lse.dtype == torch.float32
        tokens = torch.empty(3, 5, dtype=torch.int64)
        got = ops.draft_accept(tokens, None, n, tokens, n)
        assert [tuple(t.shape) for t in got] == [(3, 5), (3,), (3,), (3,)]
        assert [t.dtype for t in got] == [torch.int32, torch.int32, torch.int64, torch.int32]
        assert ops.cache_keep(cache, cache, table, n, n, nodes) is None
        assert ops.cache_bounds(cache, table, n, n, bound, bound, 3) is None
        got = ops.sparse_attention(q[:, 0], cache, cache, bound, bound, table, n, 4)
        assert [tuple(t.shape) for t in got] == [(3, 4, 64), (3, 4), (3, 2, 4)] and got[2].dtype == torch.int32


def _calls(pkg, device):
    i32 = dict(dtype=torch.int32, device=device)
    f16 = dict(dtype=torch.float16, device=device)
    cache, bound, table = torch.zeros(5, 4, 2, 64, **f16), torch.zeros(5, 2, 64, **f16), torch.zeros(3, 2, **i32)
    row, nodes = torch.zeros(3, **i32), torch.zeros(3, 5, **i32)
    tokens = torch.zeros(3, 5, dtype=torch.int64, device=device)
    return {
        pkg.DraftAttentionOp: dict(q=torch.zeros(3, 5, 4, 64, **f16), k_cache=cache, v_cache=cache.clone(),
                                   page_table=table, lengths=row, drafted=row, parents=nodes),
        pkg.DraftAcceptOp: dict(tokens=tokens, parents=nodes, drafted=row, chosen=tokens, lengths=row),
        pkg.CacheKeepOp: dict(k_cache=cache, v_cache=cache.clone(), page_table=table, lengths=row, drafted=row,
                              path=nodes),
        pkg.CacheBoundsOp: dict(k_cache=cache, page_table=table, lengths=row, counts=row, lo=bound, hi=bound.clone()),
        pkg.SparseAttentionOp: dict(q=torch.zeros(3, 4, 64, **f16), k_cache=cache, v_cache=cache.clone(), lo=bound,
                                    hi=bound.clone(), page_table=table, lengths=row, top=2)}


NAMES = ["DraftAttentionOp", "DraftAcceptOp", "CacheKeepOp", "CacheBoundsOp", "SparseAttentionOp"]


@pytest.mark.parametrize("name", NAMES)
def test_host_tensors_are_refused(pkg, name):
    op = getattr(pkg, name)
    with pytest.raises(ValueError, match="one GPU"):
        op(**_calls(pkg, "cpu")[op])


@pytest.mark.gpu
@pytest.mark.parametrize("name", NAMES)
def test_one_host_tensor_is_refused(pkg, device, name):
    op = getattr(pkg, name)
    args = _calls(pkg, device)[op]
    op(**args).launch()
    torch.cuda.synchronize()
    for key, value in args.items():
        if isinstance(value, torch.Tensor):
            with pytest.raises(ValueError, match="one GPU"):
                op(**{**args, key: value.cpu()})


@pytest.mark.gpu
def test_the_operators_refuse(pkg, device):
    """The dispatcher's operators name the status; other devices and ranks are refused before a launch."""
    pkg.torch_ops()
    ops = torch.ops.mhcpre
    a = _calls(pkg, device)
    d, s = a[pkg.DraftAttentionOp], a[pkg.SparseAttentionOp]
    with pytest.raises(RuntimeError, match="invalid shape"):
        ops.draft_attention(*d.values(), None, -1)
    with pytest.raises(RuntimeError, match="tensors on"):
        ops.draft_attention(*{**d, "parents": d["parents"].cpu()}.values())
    with pytest.raises(RuntimeError, match="must be"):
        ops.draft_attention(*{**d, "q": d["q"][0]}.values())
    with pytest.raises(RuntimeError, match="top"):
        ops.sparse_attention(*{**s, "top": 0}.values())
    with pytest.raises(RuntimeError, match="invalid shape"):
        ops.sparse_attention(*s.values(), 2, 1)


# ---- the plain implementations by hand -------------------------------------------


def test_reference_trees_by_hand():
    assert ref.paths([-1, 0, 0, 2, 9], 5) == [[0], [0, 1], [0, 2], [0, 2, 3], [4]]
    assert ref.paths(None, 3) == [[0], [0, 1], [0, 1, 2]]
    assert ref.draft_accept([[7, 3, 4, 5]], [[-1, 0, 0, 2]], [4], [[4, 9, 5, 8]], [10]) == ([[0, 2, 3, -1]], [3], [8], [9])
    assert ref.draft_accept([[7, 3]], None, [5], [[3, 6]], [1]) == ([[0, -1]], [1], [3], [1])
    k = torch.arange(8.0).view(4, 2, 1, 1)
    k2, _ = ref.cache_keep(k, k, torch.tensor([[2, 0, 3]]), torch.tensor([6]), torch.tensor([4]),
                           torch.tensor([[0, 2, 3, -1]]))
    assert k2.flatten().tolist() == [0, 6, 2, 3, 4, 5, 7, 7]


def test_reference_attention_by_hand():
    """A root with two children, each of which does not see the other, and a window of two."""
    q = torch.ones(1, 3, 1, 1, dtype=torch.float16)
    k = torch.tensor([0.0, 1.0, 2.0, 3.0]).view(2, 2, 1, 1).half()
    v = torch.tensor([1.0, 10.0, 100.0, 1000.0]).view(2, 2, 1, 1).half()
    args = (q, k, v, torch.tensor([[0, 1]]), torch.tensor([4]), torch.tensor([3]), torch.tensor([[-1, 0, 0]]), 1.0)
    w = [math.exp(x) for x in range(4)]
    out, lse, _, _ = ref.draft_attention(*args)
    for node, seen in enumerate(([0, 1], [0, 1, 2], [0, 1, 3])):
        total = sum(w[x] for x in seen)
        assert abs(float(lse[0, node, 0]) - math.log(total)) < 1e-12
        assert abs(float(out[0, node, 0, 0]) - sum(w[x] * 10.0 ** x for x in seen) / total) < 1e-9
    out, _, _, _ = ref.draft_attention(*args, window=2)
    assert abs(float(out[0, 2, 0, 0]) - (w[1] * 10 + w[3] * 1000) / (w[1] + w[3])) < 1e-9


def test_reference_selection_by_hand():
    q = torch.tensor([[[1.0, -2.0], [3.0, 1.0]]])
    lo = torch.tensor([[[0.0, -1.0]], [[0.0, 0.0]], [[-9.0, 2.0]], [[5.0, 5.0]]])
    hi = lo + 1
    # up (4, 1), down (0, -2): hi . up + lo . down = 4 + 0 + 2, 4 + 1 + 0, ...
    table = torch.tensor([[1, 0, 3, 2]])
    cols = ref.sparse_columns(q, lo, hi, table, torch.tensor([4]), 1, 2, 0, 0)
    assert cols == [[[1, 2]]]
    assert ref.sparse_columns(q, lo, hi, table, torch.tensor([4]), 1, 2, 1, 0) == [[[0, 2]]]
    assert ref.sparse_columns(q, lo, hi, table, torch.tensor([3]), 1, 2, 0, 2) == [[[1, 2]]]
    lo2, hi2 = ref.cache_bounds(torch.tensor([3.0, -1.0]).view(1, 2, 1, 1), torch.tensor([[0]]), torch.tensor([2]),
                                torch.tensor([1]), torch.full((1, 1, 1), 0.5), torch.full((1, 1, 1), 0.75), 1)
    assert (float(lo2), float(hi2)) == (-1.0, 0.75)
