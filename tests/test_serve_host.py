"""The serving operators' host side without a GPU: exports, refusals, workspace
sizes, rotary frequencies, shapes for tracing.  Phase 1 never touches device
memory, so placeholder addresses are enough."""
from __future__ import annotations

import ctypes
import math

import pytest
import torch
from torch._subclasses.fake_tensor import FakeTensorMode

import serve_ref as ref

FAKE = 0x100000
F16, BF16, F32, I32, I64, F64 = 1, 27, 0, 3, 9, 11


@pytest.fixture(scope="module")
def lib(pkg):
    return pkg.load_serve_library()


def code(pkg, name):
    return pkg.binding.STATUS_CODE["MHC_STATUS_" + name]


def strides(dims):
    out = [1]
    for d in reversed(dims[1:]):
        out.insert(0, out[0] * max(d, 1))
    return out


class S:
    """A strided tensor's description, D a dense one's; None stands for NULL."""

    def __init__(self, dims, dtype=BF16, data=FAKE, st=None):
        self.dims, self.dtype, self.data, self.st = dims, dtype, data, st

    def make(self, pkg):
        return pkg.make_strided(self.data, self.dtype, self.dims, strides(self.dims) if self.st is None else self.st)


class D(S):
    def make(self, pkg):
        return pkg.make_tensor(self.data, self.dtype, self.dims)


def call(pkg, lib, name, args):
    """(status of phase 1, workspace, status of phase 2 without a workspace where one is needed)."""
    ws, exe = ctypes.c_uint64(0), ctypes.c_void_p(None)
    made = [a.make(pkg) if isinstance(a, S) else a for a in args]
    refs = [ctypes.byref(m) if isinstance(m, ctypes.Structure) else m for m in made]
    st = getattr(lib, name + "GetWorkspaceSize")(*refs, ctypes.byref(ws), ctypes.byref(exe))
    second = None
    if st == 0 and ws.value > 0:
        launch = getattr(lib, name)
        second = [launch(None, ws.value, exe, None), launch(ctypes.c_void_p(FAKE), ws.value - 1, exe, None),
                  launch(ctypes.c_void_p(FAKE + 16), ws.value, exe, None)]
    if exe.value:
        assert lib.mhcServeExecutorDestroy(exe) == 0
    return st, int(ws.value), second


def attention(**over):
    a = dict(q=S([3, 8, 64]), k=S([20, 16, 2, 64]), v=S([20, 16, 2, 64]), table=D([3, 5], I32), lengths=D([3], I32),
             scale=0.125, window=0, out=S([3, 8, 64]), lse=D([3, 8], F32))
    assert set(over) <= set(a)
    return list({**a, **over}.values())


def rope(append=False, **over):
    a = dict(q=S([5, 4, 64]), k=S([5, 2, 64]), v=S([5, 2, 64]) if append else None, positions=D([5], I64),
             inv_freq=D([16], F64), qw=D([64], F32), kw=D([64], F32), eps=1e-6, interleaved=0, amplitude=1.0,
             slots=D([5], I64) if append else None, q_out=S([5, 4, 64]), k_out=None if append else S([5, 2, 64]),
             k_cache=S([9, 4, 2, 64]) if append else None, v_cache=S([9, 4, 2, 64]) if append else None)
    assert set(over) <= set(a)
    return list({**a, **over}.values())


def update(**over):
    a = dict(table=D([6, 7], I32), lengths=D([6], I32), parents=D([6], I32), counts=D([6], I32), pages=50, page=16,
             new_table=D([6, 7], I32), new_lengths=D([6], I32), slots=D([6, 3], I64), granted=D([6], I32),
             src=D([6], I32), dst=D([6], I32))
    assert set(over) <= set(a)
    return list({**a, **over}.values())


def compact(**over):
    a = dict(table=D([6, 7], I32), lengths=D([6], I32), pages=51, page=16, new_table=D([6, 7], I32),
             src=D([25], I32), dst=D([25], I32), used=D([1], I32))
    assert set(over) <= set(a)
    return list({**a, **over}.values())


def copy(**over):
    a = dict(k=S([20, 16, 2, 64]), v=S([20, 16, 2, 64]), src=D([3], I32), dst=D([3], I32))
    assert set(over) <= set(a)
    return list({**a, **over}.values())


OPS = {"mhcPagedAttention": attention, "mhcQkNormRope": rope, "mhcCacheUpdate": update, "mhcCacheCompact": compact,
       "mhcCacheCopyPages": copy}


def test_library_exports_every_declared_symbol(pkg, lib):
    names = pkg.exported_symbols(pkg.serve.SERVE_HEADER)
    assert set(names) >= {n + s for n in OPS for s in ("", "GetWorkspaceSize")} | {"mhcServeExecutorDestroy"}
    for name in names:
        assert hasattr(lib, name), name


@pytest.mark.parametrize("name", OPS)
def test_valid_calls_and_workspaces(pkg, lib, name):
    st, ws, second = call(pkg, lib, name, OPS[name]())
    assert st == 0
    if ws:
        assert second == [code(pkg, "WORKSPACE_TOO_SMALL")] * 3
    assert getattr(lib, name)(None, 0, None, None) == code(pkg, "NULL_ARGUMENT")


def test_an_executor_launches_its_own_operator_only(pkg, lib):
    ws, exe = ctypes.c_uint64(0), ctypes.c_void_p(None)
    made = [a.make(pkg) if isinstance(a, S) else a for a in copy(src=D([0], I32), dst=D([0], I32))]
    refs = [ctypes.byref(m) for m in made]
    assert lib.mhcCacheCopyPagesGetWorkspaceSize(*refs, ctypes.byref(ws), ctypes.byref(exe)) == 0
    assert lib.mhcQkNormRope(None, 0, exe, None) == code(pkg, "INVALID_SHAPE")
    assert lib.mhcCacheCopyPages(None, 0, exe, None) == 0  # nothing to copy: no device is needed
    assert lib.mhcServeExecutorDestroy(exe) == 0
    assert lib.mhcServeExecutorDestroy(None) == code(pkg, "NULL_ARGUMENT")


BIG = 2 ** 33
NULLS = [(n, k) for n, f in (("mhcPagedAttention", ("q", "k", "v", "table", "lengths", "out")),
                             ("mhcQkNormRope", ("q", "k", "positions", "q_out", "qw", "kw", "k_out")),
                             ("mhcCacheUpdate", ("table", "lengths", "parents", "counts", "new_table", "new_lengths",
                                                 "slots", "granted", "src", "dst")),
                             ("mhcCacheCompact", ("table", "lengths", "new_table", "src", "dst", "used")),
                             ("mhcCacheCopyPages", ("k", "v", "src", "dst"))) for k in f]


@pytest.mark.parametrize("name,key", NULLS)
def test_null_arguments(pkg, lib, name, key):
    assert call(pkg, lib, name, OPS[name](**{key: None}))[0] == code(pkg, "NULL_ARGUMENT")


@pytest.mark.parametrize("over,want", [
    (dict(q=S([8, 64])), "INVALID_SHAPE"), (dict(q=S([3, 7, 64]), out=S([3, 7, 64]), lse=D([3, 7], F32)), "INVALID_SHAPE"),
    (dict(q=S([3, 8, 96])), "INVALID_SHAPE"), (dict(out=S([3, 8, 32])), "INVALID_SHAPE"),
    (dict(q=S([3, 8, 64], F32)), "INVALID_DTYPE"), (dict(q=S([3, 8, 64], F16)), "INVALID_DTYPE"),
    (dict(v=S([20, 16, 2, 64], F16)), "INVALID_DTYPE"), (dict(v=S([19, 16, 2, 64])), "INVALID_SHAPE"),
    (dict(table=D([4, 5], I32)), "INVALID_SHAPE"), (dict(table=D([3, 5], I64)), "INVALID_DTYPE"),
    (dict(table=D([3, 0], I32)), "INVALID_SHAPE"), (dict(lengths=D([2], I32)), "INVALID_SHAPE"),
    (dict(window=-1), "INVALID_SHAPE"), (dict(k=S([0, 16, 2, 64])), "INVALID_SHAPE"),
    (dict(lse=D([3, 7], F32)), "INVALID_SHAPE"), (dict(lse=D([3, 8], F64)), "INVALID_DTYPE"),
    (dict(q=S([3, 8, 72]), k=S([20, 16, 2, 72]), v=S([20, 16, 2, 72]), out=S([3, 8, 72])), "UNSUPPORTED_SHAPE"),
    (dict(table=D([3, 2 ** 28], I32)), "UNSUPPORTED_SHAPE"), (dict(q=S([3, 8, 64], data=FAKE + 8)), "MISALIGNED"),
    (dict(k=S([20, 16, 2, 64], st=[2049, 128, 64, 1])), "MISALIGNED"),
    (dict(v=S([20, 16, 2, 64], st=[2048, 128, 64, 2])), "INVALID_SHAPE"),
    (dict(v=S([20, 16, 2, 64], st=[-2048, 128, 64, 1])), "INVALID_SHAPE"),
    (dict(v=S([20, 16, 2, 64], st=[2 ** 60, 128, 64, 1])), "INVALID_SHAPE"),
    (dict(k=S([BIG, 16, 2, 64]), v=S([BIG, 16, 2, 64])), "UNSUPPORTED_SHAPE"),
    (dict(q=S([3, 8, 64], data=0)), "NULL_ARGUMENT"), (dict(lengths=D([3], I32, 0)), "NULL_ARGUMENT"),
    (dict(lengths=D([3], I32, FAKE + 2)), "MISALIGNED"), (dict(lse=None), "SUCCESS"),
    (dict(q=S([3, 8, 64], st=[64 * 99, 64, 1])), "SUCCESS"),
    (dict(q=S([0, 8, 64], data=0), table=D([0, 5], I32, 0), lengths=D([0], I32, 0), out=S([0, 8, 64], data=0),
          lse=D([0, 8], F32, 0)), "SUCCESS")])
def test_paged_attention_arguments(pkg, lib, over, want):
    assert call(pkg, lib, "mhcPagedAttention", attention(**over))[0] == code(pkg, want)


@pytest.mark.parametrize("append,over,want", [
    (False, {}, "SUCCESS"), (True, {}, "SUCCESS"), (True, dict(v=None), "NULL_ARGUMENT"),
    (True, dict(slots=None), "NULL_ARGUMENT"), (True, dict(v_cache=None), "NULL_ARGUMENT"),
    (True, dict(k_out=S([5, 2, 64])), "NULL_ARGUMENT"), (False, dict(qw=None, kw=None), "SUCCESS"),
    (False, dict(inv_freq=None), "SUCCESS"), (False, dict(inv_freq=D([33], F64)), "INVALID_SHAPE"),
    (False, dict(inv_freq=D([16], F32)), "INVALID_DTYPE"), (False, dict(inv_freq=D([0], F64, 0)), "SUCCESS"),
    (False, dict(inv_freq=D([16], F64, FAKE + 4)), "MISALIGNED"), (False, dict(qw=D([63], F32)), "INVALID_SHAPE"),
    (False, dict(kw=D([64], BF16)), "INVALID_DTYPE"), (False, dict(positions=D([5], F32)), "INVALID_DTYPE"),
    (False, dict(positions=D([5], I32)), "SUCCESS"), (False, dict(positions=D([4], I64)), "INVALID_SHAPE"),
    (False, dict(q=S([5, 4, 64], F32)), "INVALID_DTYPE"), (False, dict(k=S([5, 2, 64], F16)), "INVALID_DTYPE"),
    (False, dict(k=S([4, 2, 64])), "INVALID_SHAPE"), (False, dict(q_out=S([5, 4, 62])), "INVALID_SHAPE"),
    (False, dict(q=S([5, 4, 63]), k=S([5, 2, 63])), "UNSUPPORTED_SHAPE"),
    (False, dict(q=S([5, 4, 1026]), k=S([5, 2, 1026])), "UNSUPPORTED_SHAPE"),
    (False, dict(q=S([5, 4, 64], data=FAKE + 1)), "MISALIGNED"), (False, dict(q=S([5, 4, 64], data=FAKE + 2)), "SUCCESS"),
    (True, dict(slots=D([5], I32)), "INVALID_DTYPE"), (True, dict(k_cache=S([9, 4, 3, 64])), "INVALID_SHAPE"),
    (True, dict(v_cache=S([9, 5, 2, 64])), "INVALID_SHAPE"), (True, dict(v=S([5, 2, 64], F16)), "INVALID_DTYPE")])
def test_qk_norm_rope_arguments(pkg, lib, append, over, want):
    assert call(pkg, lib, "mhcQkNormRope", rope(append, **over))[0] == code(pkg, want)


@pytest.mark.parametrize("over,want", [
    ({}, "SUCCESS"), (dict(pages=0), "INVALID_SHAPE"), (dict(page=0), "INVALID_SHAPE"),
    (dict(pages=2 ** 31), "UNSUPPORTED_SHAPE"), (dict(page=2 ** 30), "UNSUPPORTED_SHAPE"),
    (dict(parents=D([5], I32)), "INVALID_SHAPE"), (dict(counts=D([6], I64)), "INVALID_DTYPE"),
    (dict(slots=D([6, 3], I32)), "INVALID_DTYPE"), (dict(slots=D([6], I64)), "INVALID_SHAPE"),
    (dict(slots=D([6, 0], I64, 0)), "SUCCESS"), (dict(new_table=D([6, 8], I32)), "INVALID_SHAPE"),
    (dict(dst=D([6], I32, FAKE + 1)), "MISALIGNED"), (dict(table=D([6, 7], I32, 0)), "NULL_ARGUMENT")])
def test_cache_update_arguments(pkg, lib, over, want):
    assert call(pkg, lib, "mhcCacheUpdate", update(**over))[0] == code(pkg, want)


@pytest.mark.parametrize("over,want", [
    ({}, "SUCCESS"), (dict(pages=52), "INVALID_SHAPE"), (dict(used=D([2], I32)), "INVALID_SHAPE"),
    (dict(src=D([25], I64)), "INVALID_DTYPE"), (dict(pages=1, src=D([0], I32, 0), dst=D([0], I32, 0)), "SUCCESS")])
def test_cache_compact_arguments(pkg, lib, over, want):
    assert call(pkg, lib, "mhcCacheCompact", compact(**over))[0] == code(pkg, want)


@pytest.mark.parametrize("over,want", [
    ({}, "SUCCESS"), (dict(k=S([20, 16, 2, 64], F32), v=S([20, 16, 2, 64], F32)), "SUCCESS"),
    (dict(k=S([20, 16, 2, 64], I32), v=S([20, 16, 2, 64], I32)), "INVALID_DTYPE"),
    (dict(v=S([20, 16, 2, 32])), "INVALID_SHAPE"), (dict(dst=D([4], I32)), "INVALID_SHAPE"),
    (dict(src=D([3], I64)), "INVALID_DTYPE"), (dict(k=S([20, 16, 2, 64], data=FAKE + 1)), "MISALIGNED")])
def test_cache_copy_pages_arguments(pkg, lib, over, want):
    assert call(pkg, lib, "mhcCacheCopyPages", copy(**over))[0] == code(pkg, want)


# ---- rotary frequencies ------------------------------------------------------


def test_rotary_frequencies(pkg):
    plain = [10000.0 ** (-2 * i / 64) for i in range(32)]
    near = lambda got, want: all(abs(g - w) <= 1e-13 * abs(w) for g, w in zip(got.tolist(), want))  # noqa: E731
    f = pkg.rotary_frequencies
    assert near(f(64), plain) and f(64).dtype == torch.float64 and f(64).shape == (32,)
    assert near(f(64, kind="linear", factor=8), [x / 8 for x in plain])
    based = f(64, kind="base", factor=8).tolist()
    assert based[0] == 1 and abs(based[-1] - plain[-1] / 8) < 1e-13 * plain[-1]
    L, low, high = 8192.0, 1.0, 4.0
    want = []
    for x in plain:
        turns = L * x / (2 * math.pi)
        keep = 1.0 if turns > high else 0.0 if turns < low else (turns - low) / (high - low)
        want.append(keep * x + (1 - keep) * x / 8)
    assert near(f(64, kind="ramp", factor=8, low=low, high=high, trained_length=L), want)
    assert any(x < w for x, w in zip(want, plain)) and want[0] == plain[0]
    index = lambda turns: 64 * math.log(4096 / (2 * math.pi * turns)) / (2 * math.log(10000.0))  # noqa: E731
    a, b = max(math.floor(index(32)), 0), min(math.ceil(index(1)), 63)
    keeps = [min(max(1 - (i - a) / (b - a), 0.0), 1.0) for i in range(32)]
    want = [k * x + (1 - k) * x / 4 for k, x in zip(keeps, plain)]
    assert near(f(64, kind="index_ramp", factor=4, low=1, high=32, trained_length=4096), want)


@pytest.mark.parametrize("args", [dict(rot=0), dict(rot=3), dict(rot=8, base=1.0), dict(rot=8, base=math.nan),
                                  dict(rot=8, factor=0.0), dict(rot=2, kind="base"),
                                  dict(rot=8, kind="ramp", low=2.0, high=2.0),
                                  dict(rot=8, kind="index_ramp", trained_length=0.0)])
def test_rotary_frequencies_refuses(pkg, args):
    with pytest.raises(pkg.MhcPreError):
        pkg.rotary_frequencies(**args)


def test_rotary_frequencies_null_and_kind(pkg, lib):
    assert lib.mhcRotaryFrequencies(8, 1e4, 0, 1.0, 1.0, 4.0, 8192.0, None) == code(pkg, "NULL_ARGUMENT")
    out = (ctypes.c_double * 4)()
    assert lib.mhcRotaryFrequencies(8, 1e4, 5, 1.0, 1.0, 4.0, 8192.0, out) == code(pkg, "INVALID_SHAPE")
    with pytest.raises(ValueError):
        pkg.rotary_frequencies(8, kind="other")


# ---- tracing and host tensors -------------------------------------------------


def test_shapes_for_tracing(pkg):
    pkg.torch_ops()
    ops = torch.ops.mhcpre
    with FakeTensorMode():
        q, k = torch.empty(2, 3, 4, 64, dtype=torch.float16), torch.empty(2, 3, 2, 64, dtype=torch.float16)
        cache, table = torch.empty(9, 4, 2, 64, dtype=torch.float16), torch.empty(6, 5, dtype=torch.int32)
        n = torch.empty(6, dtype=torch.int32)
        pos, freq = torch.empty(2, 3, dtype=torch.int64), torch.empty(32, dtype=torch.float64)
        a, b = ops.qk_norm_rope(q, k, pos, freq)
        assert a.shape == q.shape and b.shape == k.shape and a.dtype == torch.float16
        assert ops.qk_norm_rope_append(q, k, k, pos, freq, pos, cache, cache).shape == q.shape
        out, lse = ops.paged_attention(q, cache, cache, table, n)
        assert out.shape == q.shape and lse.shape == (2, 3, 4) and lse.dtype == torch.float32
        new = ops.cache_update(table, n, n, n, 9, 4, 3)
        assert [tuple(t.shape) for t in new] == [(6, 5), (6,), (6, 3), (6,), (6,), (6,)] and new[2].dtype == torch.int64
        assert [tuple(t.shape) for t in ops.cache_compact(table, n, 9, 4)] == [(6, 5), (4,), (4,), (1,)]
        assert ops.cache_copy_pages(cache, cache, n, n) is None


def test_host_tensors_have_no_kernel(pkg):
    pkg.torch_ops()
    q = torch.zeros(1, 2, 64, dtype=torch.float16)
    with pytest.raises(NotImplementedError):
        torch.ops.mhcpre.qk_norm_rope(q, q, torch.zeros(1, dtype=torch.int64), None)


# ---- the oracle itself ---------------------------------------------------------


def test_reference_attention_by_hand():
    q = torch.tensor([[[1.0, 0.0]]], dtype=torch.float16)
    k = torch.tensor([[[[0.0, 5.0]], [[math.log(3.0), 1.0]]]], dtype=torch.float16)
    v = torch.tensor([[[[1.0, 2.0]], [[5.0, 6.0]]]], dtype=torch.float16)
    out, lse, _, _ = ref.attention(q, k, v, torch.tensor([[0]]), torch.tensor([2]), 1.0)
    w = math.exp(float(k[0, 1, 0, 0]))
    assert abs(float(lse) - math.log(1 + w)) < 1e-12
    assert abs(float(out[0, 0, 0]) - (1 + 5 * w) / (1 + w)) < 1e-12


def test_reference_norm_rope_by_hand():
    x = torch.tensor([[[3.0, 4.0, 1.0, 2.0]]], dtype=torch.float16)
    freq, pos = torch.tensor([math.pi / 2], dtype=torch.float64), torch.tensor([1])
    y, _ = ref.norm_rope(x, None, pos, freq, 0.0, False, 2.0)
    assert torch.allclose(y[0, 0], torch.tensor([-8.0, 6.0, 1.0, 2.0], dtype=torch.float64))
    y, _ = ref.norm_rope(x, torch.full((4,), 2.0), pos, None, 0.0, True, 2.0)
    assert torch.allclose(y[0, 0], x[0, 0].double() * 2 / math.sqrt(7.5))


def test_reference_pages_by_hand():
    """A fork whose both rows append: two private copies, pages in order, the old page free afterwards."""
    table, lengths, slots, granted, src, dst = ref.update([[1, 3], [-1, -1]], [5, 0], [0, 0], [1, 1], 6, 4, 1)
    assert table == [[1, 0], [1, 2]] and lengths == [6, 6] and slots == [[1], [9]]
    assert (src, dst) == ([3, 3], [0, 2])
    assert ref.compact(table, lengths, 6, 4) == ([[1, 0], [1, 2]], [-1] * 3, [-1] * 3, [3])
    assert ref.compact([[5, 1], [4, -1]], [8, 4], 6, 4) == ([[2, 1], [0, -1]], [4, 5, -1], [0, 2, -1], [3])
