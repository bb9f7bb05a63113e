"""Tree attention against float64 with tolerances that go by what a row sees
(``tree_helpers.Case.exact``): probabilities in two 16-bit parts in every
format and type."""

import pytest
import torch

from tree_helpers import Case

pytestmark = pytest.mark.gpu
FORMATS = ["fp8_e4m3", "int8", None]

# (nodes, query heads over two key heads, head size): up to 16 rows and up to 32
# of a key head, then 64 and more, and heads of 256
ROWS = [(5, 4, 64), (5, 12, 64), (5, 20, 64), (37, 12, 64), (1, 8, 128), (5, 12, 128), (5, 20, 128), (20, 12, 128),
        (5, 4, 256), (5, 12, 256)]


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("t,heads,d", ROWS)
def test_short_contexts(fmt, dtype, t, heads, d):
    c = Case(2, t, heads, 2, d, fmt, dtype, 16, [300, 17], seed=t + d)
    c.agrees(c.run(), floor=2.0**-24)  # operands of at least 1/2, float16's half least 2^-25
    c.cache.check()
