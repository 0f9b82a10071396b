"""qk_norm_rope and qk_norm_rope_append against a plain 64-bit implementation."""
from __future__ import annotations

import math

import pytest
import torch

import serve_ref as ref

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ops(pkg, device):
    pkg.torch_ops()
    return torch.ops.mhcpre


def _near(got, x, weight, s, what):
    want, bound = ref.norm_rope(x, weight, s["positions"], s["inv_freq"], s["eps"], s["interleaved"], s["amplitude"])
    off = (got.cpu().double() - want).abs()
    assert got.dtype == x.dtype and (off <= bound).all(), f"{what}: {(off / bound).max():.3g} of its bound"


def _state(device, T, heads, kv_heads, d, rot, dtype, norm=True, interleaved=False, amplitude=1.0, seed=0, far=5000,
           positions_dtype=torch.int64, eps=1e-6, pad=0, shift=0):
    """q, k, v views of one buffer whose rows are `pad` elements longer, `shift` elements into it."""
    g = torch.Generator().manual_seed(seed)
    width = (heads + 2 * kv_heads) * d
    qkv = torch.randn(T * (width + pad) + shift, generator=g).to(dtype).to(device)[shift:].view(T, width + pad)
    q, k, v = (t.unflatten(1, (-1, d)) for t in qkv[:, :width].split([heads * d, kv_heads * d, kv_heads * d], 1))
    return dict(q=q, k=k, v=v, positions=torch.randint(0, far, (T,), generator=g).to(positions_dtype).to(device),
                inv_freq=(10000.0 ** (-torch.arange(0, rot, 2, dtype=torch.float64) / max(rot, 1))).to(device),
                q_weight=(1 + 0.3 * torch.randn(d, generator=g)).to(device) if norm else None,
                k_weight=(1 + 0.3 * torch.randn(d, generator=g)).to(device) if norm else None, eps=eps,
                interleaved=interleaved, amplitude=amplitude)


def _plain(ops, s):
    return ops.qk_norm_rope(s["q"], s["k"], s["positions"], s["inv_freq"], s["q_weight"], s["k_weight"], s["eps"],
                            s["interleaved"], s["amplitude"])


def _run(ops, s):
    q, k = _plain(ops, s)
    _near(q, s["q"], s["q_weight"], s, "q")
    _near(k, s["k"], s["k_weight"], s, "k")
    return q, k


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("d,rot", [(128, 128), (64, 64), (128, 64), (256, 256), (256, 64), (96, 48), (96, 96), (80, 80),
                                   (192, 64), (128, 0), (128, 2), (130, 66), (6, 4), (2, 2), (1024, 1024), (72, 30),
                                   (512, 128)])
def test_sizes(ops, device, d, rot, interleaved, dtype):
    _run(ops, _state(device, 13, 5, 2, d, rot, dtype, interleaved=interleaved, seed=d + rot))


@pytest.mark.parametrize("T", [1, 2, 3, 64, 333])
@pytest.mark.parametrize("heads,kv_heads", [(1, 1), (32, 8), (3, 1), (64, 4), (7, 7)])
def test_heads_and_tokens(ops, device, T, heads, kv_heads):
    _run(ops, _state(device, T, heads, kv_heads, 128, 128, torch.bfloat16, seed=T))


@pytest.mark.parametrize("norm", [False, True])
@pytest.mark.parametrize("interleaved", [False, True])
def test_amplitude_and_no_norm(ops, device, norm, interleaved):
    _run(ops, _state(device, 9, 4, 2, 64, 32, torch.float16, norm=norm, interleaved=interleaved, amplitude=1.37))


@pytest.mark.parametrize("pad,shift", [(8, 0), (3, 0), (0, 1), (1, 7), (16, 8)])
def test_strides_and_alignment(ops, device, pad, shift):
    _run(ops, _state(device, 11, 4, 2, 128, 128, torch.bfloat16, pad=pad, shift=shift))
    _run(ops, _state(device, 11, 4, 2, 96, 40, torch.float16, pad=pad, shift=shift, interleaved=True))


@pytest.mark.parametrize("positions_dtype,far", [(torch.int32, 2 ** 31 - 1), (torch.int64, 2 ** 40)])
def test_far_positions(ops, device, positions_dtype, far):
    """The angle keeps its phase at positions far beyond what a product in 32 bits could hold.  (At 2^40 the
    definition's own angle in 64 bits is good to 2^-13; a half of that, 2^-14 of |a| + |b|, is allowed on top.)"""
    s = _state(device, 50, 4, 2, 64, 64, torch.float16, norm=False, positions_dtype=positions_dtype, far=far)
    q, _ = _plain(ops, s)
    want, bound = ref.norm_rope(s["q"], None, s["positions"], s["inv_freq"], 0, False, 1.0)
    x = s["q"].cpu().double().abs()
    pair = (x[..., :32] + x[..., 32:]).repeat(1, 1, 2)
    assert ((q.cpu().double() - want).abs() <= bound + (2.0 ** -13 * 1.5 if far > 2 ** 32 else 2.0 ** -21) * pair).all()


def test_negative_positions(ops, device):
    s = _state(device, 20, 4, 2, 64, 64, torch.float16)
    s["positions"] = -s["positions"]
    _run(ops, s)


def test_zero_large_and_tiny_rows(ops, device):
    """A row of zeros gives zeros; rows whose squares are near the ends of fp32 and the eps's side of them."""
    s = _state(device, 6, 2, 1, 128, 128, torch.bfloat16)
    s["q"][0].zero_()
    s["q"][1].mul_(2.0 ** 60)
    s["q"][2].mul_(2.0 ** -30)
    s["k"][3].zero_()
    q, k = _run(ops, s)
    assert (q[0] == 0).all() and (k[3] == 0).all()
    _run(ops, {**s, "eps": 1e-2})


def test_no_token(ops, device):
    s = _state(device, 0, 4, 2, 64, 64, torch.float16)
    q, k = _plain(ops, s)
    assert q.shape == (0, 4, 64) and k.shape == (0, 2, 64)


def test_leading_dimensions_and_no_rotation(ops, device):
    s = _state(device, 6, 4, 2, 64, 64, torch.float16)
    q, k = _plain(ops, s)
    q4, k4 = ops.qk_norm_rope(s["q"].unflatten(0, (2, 3)), s["k"].unflatten(0, (2, 3)), s["positions"].view(2, 3),
                              s["inv_freq"], s["q_weight"], s["k_weight"])
    assert torch.equal(q4.view(6, 4, 64), q) and torch.equal(k4.view(6, 2, 64), k)
    q0, _ = ops.qk_norm_rope(s["q"], s["k"], s["positions"], None, s["q_weight"], s["k_weight"])
    _near(q0, s["q"], s["q_weight"], {**s, "inv_freq": None}, "q")


def test_in_place(pkg, device):
    s = _state(device, 30, 4, 2, 128, 128, torch.bfloat16)
    q, k = s["q"].clone(), s["k"].clone()
    op = pkg.QkNormRopeOp(s["q"], s["k"], s["positions"], s["inv_freq"], s["q_weight"], s["k_weight"], q_out=s["q"],
                          k_out=s["k"])
    op.launch()
    torch.cuda.synchronize()
    _near(s["q"], q, s["q_weight"], s, "q")
    _near(s["k"], k, s["k_weight"], s, "k")


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("T,heads,kv_heads,d,rot,page,slot_major,norm", [
    (1, 32, 8, 128, 128, 16, False, True), (70, 6, 3, 64, 32, 7, True, True), (33, 8, 1, 256, 256, 1, False, False),
    (300, 4, 4, 96, 96, 64, True, True), (5, 2, 2, 130, 66, 3, False, True)])
def test_append(ops, device, T, heads, kv_heads, d, rot, page, slot_major, norm, interleaved, dtype):
    s = _state(device, T, heads, kv_heads, d, rot, dtype, norm=norm, interleaved=interleaved)
    pages = -(-T // page) + 2
    shape = (pages, page, kv_heads, d) if slot_major else (pages, kv_heads, page, d)
    caches = [torch.randn(shape, device=device).to(dtype) for _ in range(2)]
    if not slot_major:
        caches = [c.transpose(1, 2) for c in caches]
    before = [c.clone() for c in caches]
    slots = torch.randperm(pages * page, device=device)[:T]
    if T > 4:  # tokens without a slot: padding, and numbers beyond the cache
        slots[1], slots[3] = -1, pages * page
    q = ops.qk_norm_rope_append(s["q"], s["k"], s["v"], s["positions"], s["inv_freq"], slots, *caches, s["q_weight"],
                                s["k_weight"], s["eps"], interleaved, s["amplitude"])
    q0, k0 = _run(ops, s)
    assert torch.equal(q, q0)
    on = (slots >= 0) & (slots < pages * page)
    for c, b, rows in ((caches[0], before[0], k0), (caches[1], before[1], s["v"])):
        b[slots[on] // page, slots[on] % page] = rows[on]
        assert torch.equal(c, b)


def test_append_keeps_the_bits_of_values(ops, device):
    """Values are copied, not computed: NaN payloads and infinities included."""
    s = _state(device, 4, 2, 2, 64, 64, torch.bfloat16)
    bits = torch.randint(-2 ** 15, 2 ** 15, (4, 2, 64), dtype=torch.int16, device=device)
    caches = [torch.zeros(2, 4, 2, 64, dtype=torch.bfloat16, device=device) for _ in range(2)]
    ops.qk_norm_rope_append(s["q"], s["k"], bits.view(torch.bfloat16), s["positions"], s["inv_freq"],
                            torch.arange(4, device=device), *caches, s["q_weight"], s["k_weight"])
    assert torch.equal(caches[1][0].view(torch.int16), bits)


def test_nan_stays_in_its_row(ops, device):
    s = _state(device, 5, 4, 2, 128, 64, torch.float16)
    s["q"][2, 1, 100] = math.nan
    q, k = _plain(ops, s)
    bad = torch.isnan(q).any(2).cpu()
    assert bad.sum() == 1 and bad[2, 1] and not torch.isnan(k).any()


def test_stream_and_graph(pkg, device):
    s = _state(device, 17, 8, 2, 128, 128, torch.bfloat16)
    op = pkg.QkNormRopeOp(s["q"], s["k"], s["positions"], s["inv_freq"], s["q_weight"], s["k_weight"])
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    op.launch(side)
    side.synchronize()
    _near(op.q_out, s["q"], s["q_weight"], s, "q")
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        op.launch()
    for _ in range(3):
        s["positions"].random_(0, 10000)
        op.q_out.zero_()
        graph.replay()
        torch.cuda.synchronize()
        _near(op.q_out, s["q"], s["q_weight"], s, "q")
        _near(op.k_out, s["k"], s["k_weight"], s, "k")
