"""Gradients of packed batches of long and short sequences, padding and empty
places on the GPU: what a sequence gets goes by its own length."""

import pytest
import torch

from pass_helpers import packed_attention
from test_gpu_prompt import BF16, F16, Case, offsets_of
from voyager_amd import prompt

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("lengths,pad,heads,kv", [
    ([700, 40], 0, 3, 1), ([40, 1700], 0, 3, 1), ([1400, 3, 900], 5, 2, 1), ([40, 700], 0, 3, 1), ([600, 3, 40, 17, 900], 50, 2, 1), ([300], 600, 2, 2), ([2], 511, 2, 1),
    ([0, 1600, 0, 2, 511, 512, 0, 70], 0, 2, 2), ([513, 128, 600, 384, 1, 2], 3, 2, 1)])
def test_short_sequences_are_rounded_once_in_any_company(dtype, d, lengths, pad, heads, kv):
    """Sequences of fewer than 512 rows, beside long ones and rows that pad: a
    result's rounding is off by a fifth of its most, half a step, and more on
    average: 2^-11 of it in bfloat16, 2^-14 in float16.  Weights and their gradients
    in two parts are off by 2^-18 and 2^-22, float32 sums of at most 511 products by
    some 2^-20 of their magnitudes: under a quarter of it, added in squares 1.04."""
    c = Case(lengths, heads, kv, d, dtype, pad)
    ref, _ = packed_attention(c.q, c.k, c.v, c.offsets, c.scale, c.go)
    short = torch.zeros(c.packing.tokens, dtype=torch.bool)
    for a, b in zip(c.offsets, c.offsets[1:]):
        short[a:b] = b - a < 512
    short = short.cuda()
    for y, r, name in list(zip(c.run(), ref, ("output", "lse", "dq", "dk", "dv")))[2:]:
        y, r = y[short].double(), r[short]
        once = (r.to(dtype).double() - r).norm()
        assert float((y - r).norm()) <= float(once) * 1.04 + 1e-9, name


@pytest.mark.parametrize("dtype,d", [(BF16, 64), (F16, 64), (BF16, 128), (F16, 128), (BF16, 256)])
@pytest.mark.parametrize("lengths", [[600, 3, 40, 17, 900], [40, 1600], [511, 512], [5000, 30, 200]])
def test_values_and_gradients_of_mixed_batches(dtype, d, lengths):
    Case(lengths, 4, 2, d, dtype, 77).check()


@pytest.mark.parametrize("dtype,d,heads", [(BF16, 256, 2), (F16, 256, 2), (BF16, 128, 88), (F16, 64, 176)])
@pytest.mark.parametrize("lengths", [[700], [600, 100, 40]])
def test_empty_places_change_nothing(dtype, d, heads, lengths):
    """Offsets filled up to a fixed number, as a captured step has them.  (Heads of
    64 and 128: so many that no workgroup's halves share a block, which goes by the
    number of places.)"""
    c = Case(lengths, heads, 1, d, dtype, 6)
    want = c.run()
    for places in ([*lengths, *[0] * 61], [0] * 30 + lengths + [0] * 3):
        offsets = torch.tensor(offsets_of(places), dtype=torch.int32).cuda()
        c.packing = prompt.Packing(offsets, c.packing.tokens)
        assert all(torch.equal(a, b) for a, b in zip(c.run(), want))
