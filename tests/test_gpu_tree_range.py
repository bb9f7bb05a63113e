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
