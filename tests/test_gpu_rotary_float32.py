"""Float32 rotary positions: sine and cosine are right to their last bit."""

import pytest
import torch

from voyager_amd import rotary

pytestmark = pytest.mark.gpu


def _parts(x, rotary_dim, interleaved):
    part = x[..., :rotary_dim]
    return (part[..., 0::2], part[..., 1::2]) if interleaved else (part[..., : rotary_dim // 2], part[..., rotary_dim // 2:])


@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("tokens,heads,dim,rotary_dim", [(1, 3, 128, 128), (300, 2, 64, 32), (2500, 2, 128, 64), (40, 1, 10, 6)])
@pytest.mark.parametrize("scaling", [None, {"kind": "yarn", "factor": 16.0, "low": 1.0, "high": 32.0, "trained": 4096}])
def test_each_value_to_its_roundings(interleaved, tokens, heads, dim, rotary_dim, scaling):
    """y0 = x0 c - x1 s: c and s rounded once each (half a step of each term),
    one product's rounding, the difference's; 1 + 2^-10 for their products.
    The angle, up to 2^20, is a float64: turns a position and their product
    here, radians and theirs there, 2^-33 each."""
    g = torch.Generator().manual_seed(tokens)
    x = torch.randn(1, tokens, heads, dim, generator=g)
    x[..., 1::3] = 0.0  # one term alone: nothing hides what its factor is off by
    positions = torch.randint(0, 1 << 20, (tokens,), generator=g)
    r = rotary.Rotary(dim, theta=5e5, rotary_dim=rotary_dim, interleaved=interleaved, scaling=scaling)
    f, factor = rotary.frequencies(rotary_dim, 5e5, scaling)
    angle = (positions.double()[:, None] * f)[None, :, None]
    for sign in (1.0, -1.0):
        if sign > 0:
            y = r(x.cuda(), None, positions.cuda())[0].cpu()
        else:  # the gradient
            leaf = torch.zeros_like(x).cuda().requires_grad_()
            (y,) = torch.autograd.grad(r(leaf, None, positions.cuda())[0], leaf, x.cuda())
            y = y.cpu()
        c, s = angle.cos() * factor, angle.sin() * factor * sign
        (x0, x1), (y0, y1) = _parts(x.double(), rotary_dim, interleaved), _parts(y.double(), rotary_dim, interleaved)
        for got, a, b in ((y0, x0 * c, -x1 * s), (y1, x1 * c, x0 * s)):
            tol = 2.0**-24 * (1 + 2.0**-10) * ((a + b).abs() + a.abs() + b.abs() + torch.maximum(a.abs(), b.abs()))
            tol += 4 * 2.0**-33 * factor * (x0.abs() + x1.abs())
            err = (got - (a + b)).abs()
            assert bool((err <= tol).all()), f"worst {float((err / tol).max()):.1f}"
