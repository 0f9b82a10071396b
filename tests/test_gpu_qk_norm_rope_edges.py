"""qk_norm_rope where a row's mean square is below fp32's normal values."""
from __future__ import annotations

import pytest
import torch

import serve_ref as ref

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("d", [128, 130])  # the paths of 16-byte pieces and of single values
@pytest.mark.parametrize("eps", [0.0, 1e-40])
def test_tiny_rows(pkg, device, d, eps):
    """Squares of 2^-130 are whole multiples of 2^-149, each off by 2^-150 at most: together as far as 2^-18 of their
    mean, which is less than half of what the d + 8 roundings of the bound allow."""
    pkg.torch_ops()
    g = torch.Generator().manual_seed(d)
    x = (torch.randn(7, 3, d, generator=g) * 2.0 ** -65).to(torch.bfloat16).to(device)
    x[0] *= 2.0 ** 40  # ordinary ones among them
    positions, weight = torch.arange(7, device=device), (1 + 0.3 * torch.randn(d, generator=g)).to(device)
    q, k = torch.ops.mhcpre.qk_norm_rope(x, x, positions, None, weight, weight, eps)
    want, bound = ref.norm_rope(x, weight, positions, None, float(torch.tensor(eps, dtype=torch.float32)), False, 1.0)
    for y in (q, k):
        off = (y.cpu().double() - want).abs()
        assert (off <= bound).all(), f"{(off / bound).max():.3g} of its bound"
