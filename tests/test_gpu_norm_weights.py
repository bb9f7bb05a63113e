"""The norms' weights' gradients in float32 on the GPU: sums over all rows that lose little."""

import pytest
import torch

from pass_helpers import U
from voyager_amd import rotary

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("dim,tokens,heads", [(8, 64, 256), (2, 700, 256), (4, 640, 128), (8, 1000, 100), (64, 600, 32)])
def test_sums_of_equal_terms(dtype, dim, tokens, heads):
    """All rows are one row, which sums in float32 round the same way each time, off
    by up to half of their number.  A term is off by the root's squares (dim / 2 + 3 roundings) and
    6 more (no turn: position 0), a lane's sum of two terms at most by two, the sums of
    those in float64 by nothing, and the result by one."""
    rot = rotary.Rotary(dim)
    worst = 0.0
    for seed in range(12):
        g = torch.Generator().manual_seed(seed)
        x, go = (torch.rand(dim, generator=g).to(dtype).cuda() + 0.5 for _ in range(2))
        w = torch.ones(dim, device="cuda", requires_grad=True)
        rows = x.expand(1, tokens, heads, dim).contiguous()
        y, _ = rot.normed(rows, None, torch.zeros(tokens, dtype=torch.int64, device="cuda"), w, None)
        (dw,) = torch.autograd.grad(y, w, go.expand(1, tokens, heads, dim).contiguous())
        a = x.double()
        ref = tokens * heads * go.double() * a * (a.square().mean() + 1e-6) ** -0.5
        worst = max(worst, float(((dw.double() - ref) / ref).abs().max()))
    assert worst <= (dim / 2 + 3 + 6 + 2 + 1) * U, worst / U
