"""PyTorch operators ``torch.ops.mhcpre.mhc_pre`` and
``torch.ops.mhcpre.mhc_pre_with_h_pre``, and the serving operators
``qk_norm_rope``, ``qk_norm_rope_append``, ``paged_attention``,
``cache_update``, ``cache_compact``, ``cache_copy_pages``, ``draft_attention``,
``draft_accept``, ``cache_keep``, ``cache_bounds`` and ``sparse_attention``
(native too, from ``csrc/mhc_serve_torch.cpp`` over ``include/mhc_serve.h``, which
says what each computes).

The serving operators take x-like tensors as ``[..., heads, d]`` with any
leading dimensions; inputs that are not laid out as the C ABI wants them are
copied first, caches never are.

The operators are native: ``libmhcpre_torch.so`` (built from
``csrc/mhc_pre_torch.cpp``) registers them with PyTorch's dispatcher and calls
the C ABI of ``libmhcpre.so`` from C++.  They mirror the two phase-1 entry
points of the C ABI (``mhcPreGetWorkspaceSize`` and
``mhcPreGetWorkspaceSizeWithHPre``, the latter also writing hPre): each call
runs phase 1 on the given tensors, allocates the outputs and the workspace
from PyTorch's caching allocator and launches on the current stream.
Arguments, defaults and validation are those of the reference operator
(``code/op_host/mhc_pre.cpp:57-79,126-130,217-257,297-298``): x
``[..., n, D]`` fp16/bf16, phi ``[n*D, M]`` fp32 read as memory ``[M][K]``,
alpha ``[3]``, bias ``[M]``, gamma ``[n, D]`` or None.  Outputs are new
tensors: hIn ``[..., D]`` (x's dtype), hPost ``[..., n]``, hRes
``[..., n, n]`` and hPre ``[..., n]`` (fp32).  A status the library returns
is raised as RuntimeError naming it.

Only device (ROCm "cuda") tensors have a kernel; the fake implementation
registered here gives shapes and dtypes for tracing (meta / fake tensors,
torch.compile).  There is no CPU implementation and no autograd formula (the
reference operator is forward-only).

Phase 1 is cheap on a repeated shape: the library caches the plan per shape,
dtypes, gamma presence, eps and device, and each call only validates and
binds the new tensors.

Expired waits.  The persistent kernels' workgroups wait on each other with a
bound; if another kernel holds CUs they need (an RCCL kernel on a
communication stream, say), a wait can expire and the rows it was for come
out NaN.  Every executor the operators create reports such a launch in a
per-device sticky status word (mhcPreExecutorSetStatusWord): read it with
:func:`device_status` after any synchronization of your own, clear it with
:func:`clear_device_status`.  MHCPRE_CHECK_STATUS=1 instead synchronizes after
every call and raises.
"""
from __future__ import annotations

from pathlib import Path

import torch

from .binding import load_library

_LIB_NAME = "mhcpre"
_PKG_DIR = Path(__file__).resolve().parent


def library_path() -> Path:
    return _PKG_DIR / "libmhcpre_torch.so"


def _load() -> None:
    """Load the native operators.  Raises if they are not built: there is no
    Python fallback."""
    load_library()  # libmhcpre.so first (the operators' library links it in place)
    path = library_path()
    if not path.exists():
        raise FileNotFoundError(
            f"{path} not built; build it with `make -C mhcpre-review_amd/csrc torch` "
            "or __graft_entry__.build()")
    torch.ops.load_library(str(path))


_load()


def _device_index(device) -> int:
    if device is None:
        return torch.cuda.current_device()
    d = torch.device(device)
    return d.index if d.index is not None else torch.cuda.current_device()


def device_status(device=None) -> int:
    """0, or MHC_STATUS_DEVICE_TIMEOUT (8) if a launch of the operators on
    ``device`` (default: the current one) left NaN rows since the last
    :func:`clear_device_status`.  Reading the word waits for the launches
    enqueued before it on the current stream, as any read of a device tensor
    does; it adds no synchronization of the operators' own."""
    return int(torch.ops.mhcpre.status_word(_device_index(device)).item())


def clear_device_status(device=None) -> None:
    torch.ops.mhcpre.status_word(_device_index(device)).zero_()


def _fake_outputs(x):
    # The C ABI accepts x as [B, S, n, D] (the reference's layout) or [T, n, D].
    if x.dim() not in (3, 4):
        raise ValueError(f"x must be [B, S, n, D] or [T, n, D], got {tuple(x.shape)}")
    lead = tuple(x.shape[:-2])
    n, D = x.shape[-2], x.shape[-1]
    return (x.new_empty(lead + (D,)),
            x.new_empty(lead + (n,), dtype=torch.float32),
            x.new_empty(lead + (n, n), dtype=torch.float32),
            x.new_empty(lead + (n,), dtype=torch.float32))


@torch.library.register_fake(f"{_LIB_NAME}::mhc_pre")
def _(x, phi, alpha, bias, gamma=None, norm_eps=1e-6, hc_eps=1e-6):
    return _fake_outputs(x)[:3]


@torch.library.register_fake(f"{_LIB_NAME}::mhc_pre_with_h_pre")
def _(x, phi, alpha, bias, gamma=None, norm_eps=1e-6, hc_eps=1e-6):
    return _fake_outputs(x)


@torch.library.register_fake(f"{_LIB_NAME}::qk_norm_rope")
def _(q, k, positions, inv_freq, q_weight=None, k_weight=None, eps=1e-6, interleaved=False, amplitude=1.0):
    return q.new_empty(q.shape), k.new_empty(k.shape)


@torch.library.register_fake(f"{_LIB_NAME}::qk_norm_rope_append")
def _(q, k, v, positions, inv_freq, slots, k_cache, v_cache, q_weight=None, k_weight=None, eps=1e-6,
      interleaved=False, amplitude=1.0):
    return q.new_empty(q.shape)


@torch.library.register_fake(f"{_LIB_NAME}::paged_attention")
def _(q, k_cache, v_cache, page_table, lengths, scale=None, window=0):
    return q.new_empty(q.shape), q.new_empty(q.shape[:-1], dtype=torch.float32)


@torch.library.register_fake(f"{_LIB_NAME}::cache_update")
def _(page_table, lengths, parents, counts, pages, page_size, tokens=1):
    rows = page_table.shape[0]
    row = [page_table.new_empty((rows,)) for _ in range(4)]
    slots = page_table.new_empty((rows, tokens), dtype=torch.int64)
    return page_table.new_empty(page_table.shape), row[0], slots, row[1], row[2], row[3]


@torch.library.register_fake(f"{_LIB_NAME}::cache_compact")
def _(page_table, lengths, pages, page_size):
    return (page_table.new_empty(page_table.shape), page_table.new_empty((pages // 2,)),
            page_table.new_empty((pages // 2,)), page_table.new_empty((1,)))


@torch.library.register_fake(f"{_LIB_NAME}::cache_copy_pages")
def _(k_cache, v_cache, src, dst):
    return None


@torch.library.register_fake(f"{_LIB_NAME}::draft_attention")
def _(q, k_cache, v_cache, page_table, lengths, drafted, parents=None, scale=None, window=0):
    return q.new_empty(q.shape), q.new_empty(q.shape[:-1], dtype=torch.float32)


@torch.library.register_fake(f"{_LIB_NAME}::draft_accept")
def _(tokens, parents, drafted, chosen, lengths):
    rows = tokens.shape[:1]
    return (tokens.new_empty(tokens.shape, dtype=torch.int32), tokens.new_empty(rows, dtype=torch.int32),
            tokens.new_empty(rows), tokens.new_empty(rows, dtype=torch.int32))


@torch.library.register_fake(f"{_LIB_NAME}::cache_keep")
def _(k_cache, v_cache, page_table, lengths, drafted, path):
    return None


@torch.library.register_fake(f"{_LIB_NAME}::cache_bounds")
def _(k_cache, page_table, lengths, counts, lo, hi, tokens=1):
    return None


@torch.library.register_fake(f"{_LIB_NAME}::sparse_attention")
def _(q, k_cache, v_cache, lo, hi, page_table, lengths, top, first=1, last=1, scale=None):
    return (q.new_empty(q.shape), q.new_empty(q.shape[:-1], dtype=torch.float32),
            q.new_empty(q.shape[:-2] + (k_cache.shape[2], top), dtype=torch.int32))
