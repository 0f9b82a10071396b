"""ctypes binding of ``include/mhc_serve.h``: the operators that a serving step
calls between MhcPre's hIn and the attention layer's output projection.

One class per operator, as :class:`~.binding.MhcPreOp` for MhcPre: phase 1 at
construction (validation, workspace, an executor bound to the tensors), phase 2
per :meth:`launch`.  Outputs that are not given are allocated on the inputs'
device.  A status that the library returns is raised as
:class:`~.binding.MhcPreError`.
"""
from __future__ import annotations

import ctypes
from typing import Optional

from .binding import (MHC_DTYPE_BF16, MHC_DTYPE_FLOAT, MHC_DTYPE_FLOAT16, MHC_MAX_DIMS, STATUS_CODE,
                      MhcPreError, MhcTensor, _REPO_DIR, _stream_handle, load_library, make_tensor)

MHC_DTYPE_INT32 = 3
MHC_DTYPE_INT64 = 9
MHC_DTYPE_DOUBLE = 11

ROTARY_KINDS = {"plain": 0, "linear": 1, "base": 2, "ramp": 3, "index_ramp": 4}

SERVE_HEADER = _REPO_DIR / "include" / "mhc_serve.h"


class MhcStridedTensor(ctypes.Structure):
    _fields_ = [
        ("data", ctypes.c_void_p),
        ("dtype", ctypes.c_int32),
        ("ndim", ctypes.c_int32),
        ("dims", ctypes.c_int64 * MHC_MAX_DIMS),
        ("strides", ctypes.c_int64 * MHC_MAX_DIMS),
    ]


def load_serve_library() -> ctypes.CDLL:
    """libmhcpre.so with the argument types of ``mhc_serve.h`` set."""
    lib = load_library()
    if getattr(lib, "_mhc_serve_ready", False):
        return lib
    P = ctypes.POINTER
    S, T = P(MhcStridedTensor), P(MhcTensor)
    exe, size = ctypes.c_void_p, P(ctypes.c_uint64)
    i32, i64, f32, f64 = ctypes.c_int32, ctypes.c_int64, ctypes.c_float, ctypes.c_double
    out = [size, P(exe)]
    phase1 = {
        "mhcQkNormRope": [S, S, S, T, T, T, T, f32, i32, f32, T, S, S, S, S],
        "mhcPagedAttention": [S, S, S, T, T, f32, i64, S, T],
        "mhcCacheUpdate": [T, T, T, T, i64, i64, T, T, T, T, T, T],
        "mhcCacheCompact": [T, T, i64, i64, T, T, T, T],
        "mhcCacheCopyPages": [S, S, T, T],
        "mhcDraftAttention": [S, S, S, T, T, T, T, f32, i64, S, T],
        "mhcDraftAccept": [T, T, T, T, T, T, T, T, T],
        "mhcCacheKeep": [S, S, T, T, T, T],
        "mhcCacheBounds": [S, T, T, T, i64, S, S],
        "mhcSparseAttention": [S, S, S, S, S, T, T, i64, i64, i64, f32, S, T, T],
    }
    for name, args in phase1.items():
        first, second = getattr(lib, name + "GetWorkspaceSize"), getattr(lib, name)
        first.argtypes, first.restype = args + out, ctypes.c_int
        second.argtypes, second.restype = [ctypes.c_void_p, ctypes.c_uint64, exe, ctypes.c_void_p], ctypes.c_int
    lib.mhcServeExecutorDestroy.argtypes, lib.mhcServeExecutorDestroy.restype = [exe], ctypes.c_int
    lib.mhcRotaryFrequencies.argtypes = [i32, f64, i32, f64, f64, f64, f64, P(f64)]
    lib.mhcRotaryFrequencies.restype = ctypes.c_int
    lib._mhc_serve_ready = True
    return lib


def make_strided(data_ptr: int, dtype: int, dims, strides) -> MhcStridedTensor:
    t = MhcStridedTensor()
    t.data = ctypes.c_void_p(int(data_ptr)) if data_ptr else None
    t.dtype = int(dtype)
    t.ndim = len(dims)
    if t.ndim > MHC_MAX_DIMS or len(strides) != t.ndim:
        raise ValueError("dims and strides")
    for i in range(t.ndim):
        t.dims[i], t.strides[i] = int(dims[i]), int(strides[i])
    return t


def _code(dt) -> int:
    import torch

    return {torch.float32: MHC_DTYPE_FLOAT, torch.float16: MHC_DTYPE_FLOAT16, torch.bfloat16: MHC_DTYPE_BF16,
            torch.int32: MHC_DTYPE_INT32, torch.int64: MHC_DTYPE_INT64, torch.float64: MHC_DTYPE_DOUBLE}[dt]


def _dense(t) -> Optional[MhcTensor]:
    if t is None:
        return None
    if not t.is_contiguous():
        raise ValueError("tensor must be contiguous")
    return make_tensor(t.data_ptr(), _code(t.dtype), list(t.shape))


def _strided(t) -> Optional[MhcStridedTensor]:
    if t is None:
        return None
    return make_strided(t.data_ptr(), _code(t.dtype), list(t.shape), list(t.stride()))


def rotary_frequencies(rot: int, base: float = 10000.0, kind: str = "plain", factor: float = 1.0,
                       low: float = 1.0, high: float = 4.0, trained_length: float = 8192.0, device=None):
    """Inverse frequencies float64 ``[rot / 2]`` (radians per position) for the
    first ``rot`` values of a head (mhcRotaryFrequencies): ``kind`` is "plain",
    "linear", "base", "ramp" or "index_ramp", the last four stretch them for
    contexts ``factor`` times longer than the trained length."""
    import torch

    lib = load_serve_library()
    out = (ctypes.c_double * max(rot // 2, 1))()
    if kind not in ROTARY_KINDS:
        raise ValueError(f"kind {kind!r} is none of {sorted(ROTARY_KINDS)}")
    st = lib.mhcRotaryFrequencies(rot, base, ROTARY_KINDS[kind], factor, low, high, trained_length, out)
    if st != 0:
        raise MhcPreError("mhcRotaryFrequencies", st)
    return torch.tensor(list(out)[:rot // 2], dtype=torch.float64, device=device)


class _ServeOp:
    """An executor, its workspace and the tensors that it is bound to, which are
    all on one GPU (ValueError otherwise: the kernels get their addresses)."""

    _name = ""

    def _create(self, args, tensors, workspace=None):
        import torch

        self.executor = ctypes.c_void_p(None)
        self._keep = [t for t in tensors if t is not None]
        device = self._keep[0].device
        for t in self._keep + ([workspace] if workspace is not None else []):
            if not t.is_cuda or t.device != device:
                raise ValueError(f"{self._name}: tensors must be on one GPU, not on {device} and {t.device}")
        self.lib = load_serve_library()
        ws = ctypes.c_uint64(0)
        by_ref = [ctypes.byref(a) if isinstance(a, ctypes.Structure) else a for a in args]
        phase1 = getattr(self.lib, self._name + "GetWorkspaceSize")
        st = phase1(*by_ref, ctypes.byref(ws), ctypes.byref(self.executor))
        if st != 0:
            raise MhcPreError(self._name + "GetWorkspaceSize", st)
        self.workspace_size = int(ws.value)
        if workspace is None:
            workspace = torch.empty(max(self.workspace_size, 256), dtype=torch.uint8, device=device)
        elif workspace.numel() * workspace.element_size() < self.workspace_size:
            self.close()
            raise MhcPreError("workspace", STATUS_CODE["MHC_STATUS_WORKSPACE_TOO_SMALL"])
        self.workspace = workspace
        self._dev_index = device.index
        self._phase2 = getattr(self.lib, self._name)

    def launch(self, stream=None) -> None:
        """Enqueue one launch on ``stream`` (default: the current stream of the
        tensors' device)."""
        import torch

        with torch.cuda.device(self._dev_index):
            st = self._phase2(ctypes.c_void_p(self.workspace.data_ptr()), ctypes.c_uint64(self.workspace_size),
                              self.executor, ctypes.c_void_p(_stream_handle(stream)))
        if st != 0:
            raise MhcPreError(self._name, st)

    def close(self) -> None:
        if getattr(self, "executor", None) is not None and self.executor.value:
            self.lib.mhcServeExecutorDestroy(self.executor)
            self.executor = ctypes.c_void_p(None)

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass


class QkNormRopeOp(_ServeOp):
    """mhcQkNormRope on q ``[T, heads, d]`` and k ``[T, kv_heads, d]``.  Without
    ``v``, ``slots`` and the caches the keys go to ``k_out``; with them keys and
    values go to the caches."""

    _name = "mhcQkNormRope"

    def __init__(self, q, k, positions, inv_freq=None, q_weight=None, k_weight=None, eps: float = 1e-6,
                 interleaved: bool = False, amplitude: float = 1.0, v=None, slots=None, k_cache=None,
                 v_cache=None, q_out=None, k_out=None):
        import torch

        self.q_out = q_out if q_out is not None else torch.empty_like(q, memory_format=torch.contiguous_format)
        if k_out is None and k_cache is None:
            k_out = torch.empty_like(k, memory_format=torch.contiguous_format)
        self.k_out = k_out
        self._create([_strided(q), _strided(k), _strided(v), _dense(positions), _dense(inv_freq), _dense(q_weight),
                      _dense(k_weight), eps, int(interleaved), amplitude, _dense(slots), _strided(self.q_out),
                      _strided(k_out), _strided(k_cache), _strided(v_cache)],
                     [q, k, v, positions, inv_freq, q_weight, k_weight, slots, k_cache, v_cache, self.q_out, k_out])


class PagedAttentionOp(_ServeOp):
    """mhcPagedAttention on q ``[B, heads, d]``; ``out`` and ``lse`` (fp32
    ``[B, heads]``; ``lse=False``: not written) are attributes."""

    _name = "mhcPagedAttention"

    def __init__(self, q, k_cache, v_cache, page_table, lengths, scale: Optional[float] = None, window: int = 0,
                 out=None, lse=None, workspace=None):
        import torch

        self.out = out if out is not None else torch.empty_like(q, memory_format=torch.contiguous_format)
        if lse is None:
            lse = torch.empty(q.shape[:-1], dtype=torch.float32, device=q.device)
        self.lse = lse if lse is not False else None
        scale = q.shape[-1] ** -0.5 if scale is None else scale
        self._create([_strided(q), _strided(k_cache), _strided(v_cache), _dense(page_table), _dense(lengths), scale,
                      window, _strided(self.out), _dense(self.lse)],
                     [q, k_cache, v_cache, page_table, lengths, self.out, self.lse], workspace)


class CacheUpdateOp(_ServeOp):
    """mhcCacheUpdate; the new state and the step's slots and copies are the
    attributes ``new_table``, ``new_lengths``, ``slots``, ``granted``, ``src``
    and ``dst``."""

    _name = "mhcCacheUpdate"

    def __init__(self, page_table, lengths, parents, counts, pages: int, page_size: int, tokens: int = 1,
                 new_table=None, new_lengths=None, workspace=None):
        import torch

        rows, dev = page_table.shape[0], page_table.device
        i32 = dict(dtype=torch.int32, device=dev)
        self.new_table = new_table if new_table is not None else torch.empty(page_table.shape, **i32)
        self.new_lengths = new_lengths if new_lengths is not None else torch.empty(rows, **i32)
        self.slots = torch.empty((rows, tokens), dtype=torch.int64, device=dev)
        self.granted, self.src, self.dst = (torch.empty(rows, **i32) for _ in range(3))
        self._create([_dense(page_table), _dense(lengths), _dense(parents), _dense(counts), pages, page_size,
                      _dense(self.new_table), _dense(self.new_lengths), _dense(self.slots), _dense(self.granted),
                      _dense(self.src), _dense(self.dst)],
                     [page_table, lengths, parents, counts, self.new_table, self.new_lengths, self.slots, self.granted,
                      self.src, self.dst], workspace)


class CacheCompactOp(_ServeOp):
    """mhcCacheCompact; attributes ``new_table``, ``src``, ``dst`` and ``used``."""

    _name = "mhcCacheCompact"

    def __init__(self, page_table, lengths, pages: int, page_size: int, workspace=None):
        import torch

        i32 = dict(dtype=torch.int32, device=page_table.device)
        self.new_table = torch.empty(page_table.shape, **i32)
        self.src, self.dst = torch.empty(pages // 2, **i32), torch.empty(pages // 2, **i32)
        self.used = torch.empty(1, **i32)
        self._create([_dense(page_table), _dense(lengths), pages, page_size, _dense(self.new_table), _dense(self.src),
                      _dense(self.dst), _dense(self.used)],
                     [page_table, lengths, self.new_table, self.src, self.dst, self.used], workspace)


class CopyPagesOp(_ServeOp):
    """mhcCacheCopyPages: pages src[i] of both caches to pages dst[i]."""

    _name = "mhcCacheCopyPages"

    def __init__(self, k_cache, v_cache, src, dst):
        self._create([_strided(k_cache), _strided(v_cache), _dense(src), _dense(dst)], [k_cache, v_cache, src, dst])


class DraftAttentionOp(_ServeOp):
    """mhcDraftAttention on q ``[B, S, heads, d]``: a tree of drafted tokens
    (``parents`` int32 ``[B, S]``) or a chain (None).  ``out`` and ``lse`` (fp32
    ``[B, S, heads]``; ``lse=False``: not written) are attributes."""

    _name = "mhcDraftAttention"

    def __init__(self, q, k_cache, v_cache, page_table, lengths, drafted, parents=None, scale: Optional[float] = None,
                 window: int = 0, out=None, lse=None, workspace=None):
        import torch

        self.out = out if out is not None else torch.empty_like(q, memory_format=torch.contiguous_format)
        if lse is None:
            lse = torch.empty(q.shape[:-1], dtype=torch.float32, device=q.device)
        self.lse = lse if lse is not False else None
        scale = q.shape[-1] ** -0.5 if scale is None else scale
        self._create([_strided(q), _strided(k_cache), _strided(v_cache), _dense(page_table), _dense(lengths),
                      _dense(drafted), _dense(parents), scale, window, _strided(self.out), _dense(self.lse)],
                     [q, k_cache, v_cache, page_table, lengths, drafted, parents, self.out, self.lse], workspace)


class DraftAcceptOp(_ServeOp):
    """mhcDraftAccept on tokens ``[B, S]``; attributes ``path``, ``accepted``,
    ``next`` and ``new_lengths``."""

    _name = "mhcDraftAccept"

    def __init__(self, tokens, parents, drafted, chosen, lengths):
        import torch

        i32 = dict(dtype=torch.int32, device=tokens.device)
        rows = tokens.shape[0]
        self.path = torch.empty(tokens.shape, **i32)
        self.accepted, self.new_lengths = torch.empty(rows, **i32), torch.empty(rows, **i32)
        self.next = torch.empty(rows, dtype=tokens.dtype, device=tokens.device)
        self._create([_dense(tokens), _dense(parents), _dense(drafted), _dense(chosen), _dense(lengths),
                      _dense(self.path), _dense(self.accepted), _dense(self.next), _dense(self.new_lengths)],
                     [tokens, parents, drafted, chosen, lengths, self.path, self.accepted, self.next,
                      self.new_lengths])


class CacheKeepOp(_ServeOp):
    """mhcCacheKeep: the tokens of ``path`` to the places behind the context."""

    _name = "mhcCacheKeep"

    def __init__(self, k_cache, v_cache, page_table, lengths, drafted, path):
        self._create([_strided(k_cache), _strided(v_cache), _dense(page_table), _dense(lengths), _dense(drafted),
                      _dense(path)], [k_cache, v_cache, page_table, lengths, drafted, path])


class CacheBoundsOp(_ServeOp):
    """mhcCacheBounds: ``lo`` and ``hi`` ``[pages, kv_heads, d]`` of the pages with
    the rows' last ``counts`` tokens, ``tokens`` at most."""

    _name = "mhcCacheBounds"

    def __init__(self, k_cache, page_table, lengths, counts, lo, hi, tokens: int = 1):
        self._create([_strided(k_cache), _dense(page_table), _dense(lengths), _dense(counts), tokens, _strided(lo),
                      _strided(hi)], [k_cache, page_table, lengths, counts, lo, hi])


class SparseAttentionOp(_ServeOp):
    """mhcSparseAttention on q ``[B, heads, d]``; ``out``, ``lse`` (as for
    :class:`PagedAttentionOp`) and ``columns`` int32 ``[B, kv_heads, top]`` are
    attributes."""

    _name = "mhcSparseAttention"

    def __init__(self, q, k_cache, v_cache, lo, hi, page_table, lengths, top: int, first: int = 1, last: int = 1,
                 scale: Optional[float] = None, out=None, lse=None, workspace=None):
        import torch

        self.out = out if out is not None else torch.empty_like(q, memory_format=torch.contiguous_format)
        if lse is None:
            lse = torch.empty(q.shape[:-1], dtype=torch.float32, device=q.device)
        self.lse = lse if lse is not False else None
        self.columns = torch.empty((q.shape[0], k_cache.shape[2], top), dtype=torch.int32, device=q.device)
        scale = q.shape[-1] ** -0.5 if scale is None else scale
        self._create([_strided(q), _strided(k_cache), _strided(v_cache), _strided(lo), _strided(hi),
                      _dense(page_table), _dense(lengths), top, first, last, scale, _strided(self.out),
                      _dense(self.lse), _dense(self.columns)],
                     [q, k_cache, v_cache, lo, hi, page_table, lengths, self.out, self.lse, self.columns], workspace)
