"""Tree attention where values are far apart: what a row does not see leaves
its bits."""

import pytest
import torch

from tree_helpers import Case

pytestmark = pytest.mark.gpu
FORMATS = ["fp8_e4m3", "int8", None]

# (nodes, query heads over two key heads, head size): up to 16 rows and up to 32
# of a key head, then 64 and more, and heads of 256
ROWS = [(5, 4, 64), (5, 12, 128), (5, 20, 64), (20, 12, 128), (5, 4, 256), (5, 12, 256)]


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("t,heads,d", ROWS)
@pytest.mark.parametrize("where", ["behind", "branch", "padding"])
@pytest.mark.parametrize("size", [2.0**30, 1e4])
def test_large_values_that_a_row_does_not_see_leave_its_bits(fmt, dtype, t, heads, d, where, size):
    """A row of values ``size`` times the others: behind the sequence, in
    another branch, under a node that pads."""
    if dtype == torch.float16 and size > 1e4:
        size = 2.0**13
    kv, ctx = 2, 55
    parents = torch.tensor([[-1, 0, 0, 1, 0] + [3] * (t - 5)], dtype=torch.int32)
    if where == "padding":
        parents[0, 2] = -1
    c = Case(1, t, heads, kv, d, fmt, dtype, 16, [ctx], seed=t + d, spread=0.0, parents=parents)
    clean = c.run()
    at = ctx + (t if where == "behind" else 2)
    c.v[0, at] = (c.v[0, at].float() * size).to(dtype)
    c.fill()
    o, lse = c.run()
    others = ~c.see[0, :, 2] if where == "branch" else torch.ones(t, dtype=torch.bool)
    assert torch.equal(o[0, others], clean[0][0, others]), "rows that do not see it changed"
    assert torch.equal(lse, clean[1])


# One to 32768 others: up to 16 rows and up to 32 of a key head, then 64, more, and heads of 256
SINKS = [(1, 4, 64), (3, 8, 128), (10, 4, 64), (20, 8, 128), (1, 4, 256), (5, 8, 256)]


def _beside(fmt, dtype, t, heads, d, nats, others, first, seed):
    """A key ``nats`` above all others of value ``first``; theirs are near 1."""
    c = Case(1, t, heads, 1, d, fmt, dtype, 64, [others], seed=seed, spread=0.0, parents=None)
    g = torch.Generator().manual_seed(seed)
    base = torch.randn(d, generator=g)
    base *= (d ** 0.5) / base.norm()  # score of base and base: d ** 0.5
    c.q = (base + 0.05 * torch.randn(1, t, heads, d, generator=g)).to(dtype).cuda()
    c.k = (0.01 * torch.randn(c.k.shape, generator=g)).to(dtype).cuda()
    c.k[0, 0, 0] = (base * nats / d ** 0.5).to(dtype).cuda()
    c.v = (1 + 0.25 * torch.randn(c.v.shape, generator=g)).to(dtype).cuda()
    c.v[0, 0, 0] = (first * torch.randn(d, generator=g)).to(dtype).cuda()
    c.fill()
    return c


@pytest.mark.parametrize("fmt,dtype", [("fp8_e4m3", torch.bfloat16), ("int8", torch.bfloat16), ("int8", torch.float16),
                                       ("fp8_e4m3", torch.float16), (None, torch.bfloat16), (None, torch.float16)])
@pytest.mark.parametrize("t,heads,d", SINKS)
def test_many_keys_of_little_probability_beside_one(fmt, dtype, t, heads, d):
    """The first key takes nearly all of the sum and has a small value, as
    first tokens often do: the others, each 2^-26 of it, are half of the
    result."""
    c = _beside(fmt, dtype, t, heads, d, 18.0, 32768, 2.0**-11, seed=t)
    c.agrees(c.run(), floor=2.0**-34)
    c.agrees(c.run(workgroups=4), floor=2.0**-34)


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("t,heads,d", SINKS)
def test_a_large_value_of_next_to_no_probability(fmt, t, heads, d):
    c = _beside(fmt, torch.bfloat16, t, heads, d, -70.0, 300, 2.0**40, seed=t)
    c.agrees(c.run(), floor=2.0**-34)
    c.agrees(c.run(workgroups=1), floor=2.0**-34)


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("rising", [1, -1])
@pytest.mark.parametrize("t,heads,d", SINKS)
def test_values_over_many_binades(fmt, t, heads, d, rising):
    """Values that grow, or shrink, a binade every 12 keys."""
    c = Case(1, t, heads, 1, d, fmt, torch.bfloat16, 64, [640], seed=t, spread=0.0, parents=None)
    at = torch.arange(c.v.shape[1]).cuda()[:, None, None] / 12.0
    c.v = (c.v.float() * torch.exp2(rising * at)).bfloat16()
    c.fill()
    for workgroups in (0, 1):
        c.agrees(c.run(workgroups=workgroups), floor=2.0**-34)


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("t,heads,d", SINKS)
@pytest.mark.parametrize("size", [2.0**126, 2.0**-80])
def test_values_near_the_ends_of_their_type(fmt, t, heads, d, size):
    """Values between 1 and 2 times ``size`` under scores that grow along the
    keys: sums of exponentials times such values are not finite, results are."""
    c = Case(2, t, heads, 1, d, fmt, torch.bfloat16, 64, [1500, 70], seed=t, spread=0.0, parents=None)
    g = torch.Generator().manual_seed(t)
    at = torch.arange(c.k.shape[1])[:, None, None]
    base = torch.randn(d, generator=g)
    base *= d ** 0.5 / base.norm()
    c.q = (base + 0.1 * torch.randn(c.q.shape, generator=g)).bfloat16().cuda()
    c.k = (base * at * 0.004 / d ** 0.5 + 0.3 * torch.randn(c.k.shape, generator=g)).bfloat16().cuda()
    c.v = ((1 + 0.9 * torch.rand(c.v.shape, generator=g)) * size).bfloat16().cuda()
    c.fill()
    for workgroups in (0, 1, 8):
        c.agrees(c.run(workgroups), floor=2.0**-34)
