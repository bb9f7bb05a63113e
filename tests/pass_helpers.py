"""Plain forms, in float64, of the operators of a pass over packed sequences:
norms with rotary positions, causal attention, scores of given tokens."""

import math

import torch

from draft_helpers import HALF, turned

U = 2.0**-24  # half a step of float32, relative


# ------------------------------------------------------- norms and positions
def spread(x, rotary, interleaved):
    """|x0| + |x1| of every pair, and |x| of the channels that do not turn."""
    m = x.double().abs().clone()
    part = m[..., :rotary].clone()
    if interleaved:
        s = part[..., 0::2] + part[..., 1::2]
        m[..., :rotary] = torch.stack((s, s), -1).flatten(-2)
    else:
        s = part[..., : rotary // 2] + part[..., rotary // 2:]
        m[..., :rotary] = torch.cat((s, s), -1)
    return m


def norm_turned(x, w, positions, freq, factor, rotary, interleaved, eps):
    """``(y, tolerance)``.  r: dim squares summed (half of that in the root) and
    three roundings; two products; then the turn's 10 roundings as for
    vh_rope; half a step of the result, which has a least size."""
    a, dim = x.double(), x.shape[-1]
    z = a * (a.square().mean(-1, keepdim=True) + eps) ** -0.5 * w.double()
    y = turned(z, positions, freq, factor, rotary, interleaved)
    tol = HALF[x.dtype] * y.abs() + (dim / 2 + 15) * U * factor * spread(z, rotary, interleaved) + least(x.dtype)
    return y, tol


def least(dtype):
    """Half of the least step of a type."""
    f = torch.finfo(dtype)
    return f.smallest_normal * f.eps / 2


def norm_turned_back(x, w, g, positions, freq, factor, rotary, interleaved, eps):
    """``(dx, dw, tolerance of dx, tolerance of dw)`` for the result's gradient
    g: the turn back (10 roundings of a pair's magnitudes), r as above, products
    and a sum of dim terms; for dw a sum over all rows."""
    a, dim = x.double(), x.shape[-1]
    r = (a.square().mean(-1, keepdim=True) + eps) ** -0.5
    z = a * r
    back = turned(g.double(), positions, freq, factor, rotary, interleaved, back=True)
    size = factor * spread(g, rotary, interleaved)
    b, bm = back * w.double(), size * w.double().abs()
    dx = r * (b - z * (b * z).mean(-1, keepdim=True))
    c = (dim + 24) * U
    tol = HALF[x.dtype] * dx.abs() + c * r * (bm + z.abs() * 2 * (bm * z.abs()).mean(-1, keepdim=True)) + least(x.dtype)
    rows = (0, 1, 2)
    dw = (back * z).sum(rows)
    n = x.shape[0] * x.shape[1] * x.shape[2]
    tw = HALF[w.dtype] * dw.abs() + (c + n * U) * (size * z.abs()).sum(rows) + least(w.dtype)
    return dx, dw, tol, tw


def within(got, ref, tol, what=""):
    err = (got.detach().double().cpu() - ref.cpu()).abs()
    ok = (err <= tol.cpu()) | (torch.isnan(ref.cpu()) & torch.isnan(err))
    assert bool(ok.all()), f"{what}: {int((~ok).sum())} of {ok.numel()} beyond, worst {float((err / tol.cpu()).max()):.3g}"
