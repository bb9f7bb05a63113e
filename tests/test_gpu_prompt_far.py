"""Attention of far scores on the GPU: a row's logarithm of a sum is a large
float32 number, whose rounding has to have no part in the weights."""

import pytest
import torch

from pass_helpers import U, least, within
from draft_helpers import HALF
from test_gpu_prompt import BF16, F16, Case

pytestmark = pytest.mark.gpu
LENGTHS = [[40], [300, 7], [700], [900, 40]]


@pytest.mark.parametrize("dtype,d", [(BF16, 64), (F16, 64), (BF16, 128), (F16, 128), (BF16, 256), (F16, 256)])
@pytest.mark.parametrize("scale", [1.0, 16.0])
@pytest.mark.parametrize("lengths", LENGTHS)
def test_values_gradient_of_far_keys(dtype, d, scale, lengths):
    """Each row is its own key's alone, with a score of 2^13 or 2^17: it gives that
    key's value its gradient as it is.  A weight is off from 1 by the logarithm's
    and the power's 2^-20 (scores are the same in both passes), under half a
    step of 16 bits, and so the gradient is the one given."""
    c = Case(lengths, 2, 2, d, dtype, scale=scale)
    c.k = (8192 ** 0.5 * torch.nn.functional.normalize(c.k.float(), dim=2)).to(dtype)
    _, lse, _, _, dv = c.run(q=c.k)
    assert 8000 * scale < float(lse.min()) and float(lse.max()) < 8400 * scale
    assert torch.equal(dv, c.go)


@pytest.mark.parametrize("dtype,d", [(BF16, 64), (F16, 64), (BF16, 128), (F16, 128), (BF16, 256), (F16, 256)])
@pytest.mark.parametrize("scale", [1.0, 16.0])
@pytest.mark.parametrize("lengths", LENGTHS)
def test_values_gradient_of_equal_far_keys(dtype, d, scale, lengths):
    """All keys of a sequence are one: row i (from 0 on) gives each of its keys the (i + 1)-th
    part.  Scores are equal bit for bit; a weight is off by 2^-20 of it, by its
    rounding, half a step (of two parts 2^-17 at most), and sums of n terms by n 2^-24; float16's least
    weight, lifted by 2^15, is 2^-39."""
    c = Case(lengths, 2, 2, d, dtype, scale=scale)
    one = (8192 ** 0.5 * torch.nn.functional.normalize(c.k[:1].float(), dim=2)).to(dtype)
    c.k = c.q = one.expand(c.k.shape).contiguous()
    dv = c.run()[4]
    ref, tol = torch.zeros_like(dv, dtype=torch.float64), torch.zeros_like(dv, dtype=torch.float64)
    for a, b in zip(c.offsets, c.offsets[1:]):
        n = b - a
        part = c.go[a:b].double() / torch.arange(1, n + 1, device="cuda").double()[:, None, None]
        back = lambda x: x.flip(0).cumsum(0).flip(0)
        ref[a:b] = back(part)
        each = 2.0**-20 + (n + 64) * U + (2.0**-17 if n < 512 else HALF[dtype])
        tol[a:b] = each * back(part.abs()) + HALF[dtype] * ref[a:b].abs() * 1.01 + least(dtype)
        if dtype == F16:
            tol[a:b] += 2.0**-39 * back(c.go[a:b].double().abs())
    within(dv, ref, tol, "dv")
