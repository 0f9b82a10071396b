"""draft_attention with finite values near the end of bf16, whose sums pass the end of fp32 unless they are scaled."""
from __future__ import annotations

import math

import pytest
import torch

import draft_ref as ref
from test_gpu_draft_attention import BF16, check, make, ops  # noqa: F401

pytestmark = pytest.mark.gpu
MOST = torch.finfo(BF16).max

# Rows of a kv head for each layout, and heads of one padded and one of two loads.
LAYOUTS = [(3, 8, 2, 64), (25, 4, 2, 128), (50, 2, 1, 80), (100, 2, 1, 64), (150, 4, 2, 128), (12, 4, 1, 256)]


def _put(a, row, token, head, value, dim=slice(None)):
    page = a["v_cache"].shape[1]
    a["v_cache"][int(a["page_table"][row, token // page]), token % page, head, dim] = value


@pytest.mark.parametrize("S,heads,kv_heads,d", LAYOUTS)
@pytest.mark.parametrize("longest", [300, 3000])
def test_values_of_any_size(ops, device, S, heads, kv_heads, d, longest):  # noqa: F811
    """All values a quarter to all of the type's largest, of both signs, in one part and in several."""
    a = make(device, 2, S, heads, kv_heads, d, 16, longest, BF16, lengths=[longest, longest - 40], drafted=[S, S])
    g = torch.Generator(device=device).manual_seed(d)
    size = 0.25 + 0.75 * torch.rand(a["v_cache"].shape, generator=g, device=device)
    sign = torch.where(torch.isnan(a["v_cache"]), math.nan, torch.sign(a["v_cache"]))
    a["v_cache"].copy_((size * sign * (MOST / 256)).to(BF16) * 256)
    check(ops, a)


@pytest.mark.parametrize("S,heads,kv_heads,d", LAYOUTS)
def test_equal_values_come_out_as_they_are(ops, device, S, heads, kv_heads, d):  # noqa: F811
    """The mean of the largest value there is: weights and their sum are off by less than 2^-15, half the type's step
    is 2^-9 of it."""
    a = make(device, 1, S, heads, kv_heads, d, 16, 2000, BF16, lengths=[2000], drafted=[S])
    a["v_cache"].copy_(torch.where(torch.isnan(a["v_cache"]), math.nan, MOST))
    out, _ = check(ops, a)
    assert (out == MOST).all()


@pytest.mark.parametrize("S,heads,kv_heads,d", LAYOUTS)
@pytest.mark.parametrize("nats", [0.5, 2.0, 3.4])
def test_a_large_value_behind_a_lower_maximum(ops, device, S, heads, kv_heads, d, nats):  # noqa: F811
    """2e37 at a key whose score lies up to 3.4 above those before it: a reference that follows the maximum with slack
    gives it a weight above 1.  The same sequence 300 times, so that a workgroup goes over many of its tiles."""
    a = make(device, 1, S, heads, kv_heads, d, 16, 500, BF16, lengths=[500], drafted=[S])
    a["q"].zero_()
    a["q"][..., 0] = 1
    for t in range(500):
        page = int(a["page_table"][0, t // 16])
        a["k_cache"][page, t % 16, :, 0] = nats if t >= 330 else 0.0
    _put(a, 0, 5, slice(None), -2e37, 3)
    _put(a, 0, 335, slice(None), 2e37, 3)
    _put(a, 0, 331, slice(None), 1.5e38, d - 1)
    check(ops, a, scale=1.0)
    want, want_lse, bound, lse_bound = ref.draft_attention(
        **{{"page_table": "table"}.get(k, k): v for k, v in a.items()}, scale=1.0)
    for key in ("q", "page_table", "lengths", "drafted", "parents"):
        a[key] = a[key].expand(300, *a[key].shape[1:]).contiguous()
    out, lse = (t.cpu().double() for t in ops.draft_attention(*a.values(), 1.0))
    assert torch.isfinite(out).all()
    assert ((out - want).abs() <= bound).all() and ((lse - want_lse).abs() <= lse_bound).all()


@pytest.mark.parametrize("S,heads,kv_heads,d", LAYOUTS)
def test_large_and_infinite_values_in_one_block(ops, device, S, heads, kv_heads, d):  # noqa: F811
    """Nodes that see neither keep their bits; those that see an infinite value have it in its dimension and the sums
    of the large ones in theirs."""
    a = make(device, 1, S, heads, kv_heads, d, 16, 400, BF16, lengths=[400], drafted=[S])
    plain, plain_lse = check(ops, a)
    c, big, inf = 400 - S, S // 3, S - 1
    for node in (big, inf):
        _put(a, 0, c + node, slice(None), 3e38, 3)
    paths = ref.paths(a["parents"][0].tolist(), S)
    sees_big = torch.tensor([big in p or inf in p for p in paths])
    want, want_lse = check(ops, a)
    rows = ~sees_big
    assert torch.equal(want[0, rows], plain[0, rows]) and torch.equal(want_lse[0, rows], plain_lse[0, rows])
    _put(a, 0, c + inf, slice(None), math.inf, 7)  # (the last node is nobody's ancestor)
    out, lse = (t.cpu().double() for t in ops.draft_attention(*a.values()))
    assert (out[0, inf, :, 7] == math.inf).all()
    assert torch.equal(out[0, :inf], want[0, :inf]) and torch.equal(lse[0, :inf], want_lse[0, :inf])
    others = [e for e in range(d) if e != 7]
    # (weights of 16 bits in both, rounded to 8: a step of the type at most)
    assert ((out - want)[0, inf][:, others].abs() <= 2.0 ** -7 * want[0, inf][:, others].abs() + 2.0 ** -12).all()


@pytest.mark.parametrize("bits", [108, 114, 118, 122, 126])
def test_many_parts_of_large_values(ops, device, bits):  # noqa: F811
    """One sequence over all workgroups, values of 2^bits to 3 times that: at some size each part's sum is finite and
    the sum of all is not."""
    a = make(device, 1, 3, 4, 1, 64, 64, 33000, BF16, lengths=[33000], drafted=[3])
    a["v_cache"].copy_((1 + a["v_cache"].float().abs().clamp(max=2)) * 2.0 ** bits)
    check(ops, a)


def test_small_weights_beside_large_values(ops, device):  # noqa: F811
    """A weight of e^-40 whose value is the type's largest, in a row whose other values are 1 and in one whose others are
    as large."""
    a = make(device, 2, 4, 2, 1, 64, 16, 200, BF16, lengths=[200, 200], drafted=[4, 4])
    a["q"].zero_()
    a["q"][..., 0] = 1
    a["k_cache"][..., 0] = 0
    a["v_cache"].fill_(1.0)
    a["v_cache"][a["page_table"][1].long()] = MOST / 2
    for row in range(2):
        page = int(a["page_table"][row, 2])
        a["k_cache"][page, 3, 0, 0] = -40
        a["v_cache"][page, 3, 0] = MOST
    check(ops, a, scale=1.0)
