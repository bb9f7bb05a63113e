"""Tree attention against float64 with tolerances that go by what a row sees
(``tree_helpers.Case.exact``): probabilities in two 16-bit parts in every
format and type."""

import pytest
import torch

from tree_helpers import Case
from voyager_amd import speculative

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


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("t,heads,d", ROWS)
@pytest.mark.parametrize("workgroups", [1, 40])
def test_long_splits(fmt, dtype, t, heads, d, workgroups):
    """A sequence is one split, or a few: up to 50 steps of a wave, odd ends."""
    c = Case(4, t, heads, 2, d, fmt, dtype, 32, [1601, 129, 0, 800], seed=t + d)
    c.agrees(c.run(workgroups))
    c.cache.check()


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("t,heads,d", ROWS)
@pytest.mark.parametrize("workgroups", [1, 6])
@pytest.mark.parametrize("step", [0.02, 0.2])
def test_scores_that_rise(fmt, t, heads, d, workgroups, step):
    """Scores rise by ``step`` a key and values by a binade every 40, so that
    steps of the quick form are given up in mid-loop: now and then, or each."""
    c = Case(1, t, heads, 2, d, fmt, torch.bfloat16, 16, [1100], seed=t + d, spread=0.0)
    g = torch.Generator().manual_seed(3)
    base = torch.randn(d, generator=g)
    base *= d ** 0.5 / base.norm()
    at = torch.arange(c.k.shape[1])[:, None, None]
    c.q = (base + 0.1 * torch.randn(c.q.shape, generator=g)).to(c.dtype).cuda()
    c.k = (base * at * step / d ** 0.5 + 0.1 * torch.randn(c.k.shape, generator=g)).to(c.dtype).cuda()
    c.v = (c.v.float() * torch.exp2(at.cuda() / 40.0 - 13)).to(c.dtype)
    c.fill()
    c.agrees(c.run(workgroups))


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("t,heads,d", ROWS)
@pytest.mark.parametrize("page", [16, 64])
def test_a_page_that_is_not_there_in_mid_sequence(fmt, t, heads, d, page):
    c = Case(1, t, heads, 2, d, fmt, torch.bfloat16, page, [1000], seed=t + d)
    gone = torch.zeros(1, c.k.shape[1], dtype=torch.bool)
    for at in (5, 6, 11):
        c.table[0, at] = -1 if at == 6 else c.cache.pages
        gone[0, at * page:(at + 1) * page] = True
    for workgroups in (1, 4):
        c.agrees(c.run(workgroups), gone=gone)
        with pytest.raises(RuntimeError, match="not there"):
            c.cache.check()


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("t,heads,d", [(1, 4, 64), (5, 20, 64)])
def test_more_than_a_wave_of_sequences(fmt, t, heads, d):
    """130 sequences: what a wave's lanes hold of them is scanned three times."""
    g = torch.Generator().manual_seed(4)
    contexts = torch.randint(0, 500, (130,), generator=g).tolist()
    contexts[64], contexts[129], contexts[3] = 2000, 1500, 0
    c = Case(130, t, heads, 2, d, fmt, torch.bfloat16, 16, contexts, seed=5)
    first = c.run()
    c.agrees(first)
    c.agrees(c.run(workgroups=1))
    for sequence in (63, 64, 65, 128, 129):  # each is what it is alone
        at = slice(sequence, sequence + 1)
        tree = speculative.Tree(c.parents[at].cuda())
        o, lse = speculative.tree_attention(c.q[at], c.cache, c.table[at], c.context[at], tree, return_lse=True)
        _, _, tol, tlse = c.exact()
        assert bool(((o.double() - first[0][at].double()).abs() <= 2 * tol[at]).all())
        assert bool(((lse.double() - first[1][at].double()).abs() <= 2 * tlse[at]).all())


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("b,t,heads,kv,d,context", [(2, 257, 4, 2, 64, [700, 3]), (1, 1024, 2, 1, 128, [300]),
                                                    (1, 1000, 2, 2, 256, [33])])
def test_trees_of_many_nodes(fmt, b, t, heads, kv, d, context):
    c = Case(b, t, heads, kv, d, fmt, torch.bfloat16, 16, context, seed=6)
    c.tree.check()
    c.agrees(c.run())


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("b,t,heads,kv,d,context", [(1, 513, 8, 2, 128, [1111]), (2, 1500, 8, 8, 64, [0, 40]),
                                                    (1, 4096, 4, 1, 64, [0]), (1, 700, 4, 2, 256, [300])])
def test_prompts_without_a_tree(fmt, b, t, heads, kv, d, context):
    """Row blocks by the hundred: more than the workgroups that keys are
    shared out to, so that each sequence is one split."""
    c = Case(b, t, heads, kv, d, fmt, torch.bfloat16, 64, context, seed=7, parents=None)
    c.agrees(c.run())
    c.cache.check()


@pytest.mark.parametrize("t,heads,d", ROWS)
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_infinite_values_in_mid_sequence(dtype, t, heads, d):
    """A 16-bit value that is infinite or NaN makes its channel so for the rows
    that see it, and no other."""
    c = Case(1, t, heads, 2, d, None, dtype, 16, [900], seed=t + d, spread=0.0)
    for workgroups in (1, 4):
        clean, lse = c.run(workgroups)
        was = c.v.clone()
        c.v[0, 411, 0, 3], c.v[0, 98, 0, 9], c.v[0, 700, 0, 17] = torch.inf, -torch.inf, torch.nan
        c.v[0, 50, 0, 20], c.v[0, 51, 0, 20] = torch.inf, -torch.inf
        c.fill()
        o, bad = c.run(workgroups)
        c.v = was
        c.fill()
        group = heads // 2
        head = o[0, :, :group]
        assert torch.equal(o[0, :, group:], clean[0, :, group:]) and torch.equal(bad[..., group:], lse[..., group:])
        assert bool((head[..., 3] == torch.inf).all()) and bool((head[..., 9] == -torch.inf).all())
        assert bool(torch.isnan(head[..., 17]).all()) and bool(torch.isnan(head[..., 20]).all())
        rest = [i for i in range(d) if i not in (3, 9, 17, 20)]
        ref, rlse, tol, tlse = c.exact()
        err = (head.double() - ref[0, :, :group]).abs()[..., rest]
        assert bool((err <= tol[0, :, :group][..., rest]).all())
        assert bool(((bad.double() - rlse).abs() <= tlse).all())


@pytest.mark.parametrize("fmt", ["fp8_e4m3", "int8"])
@pytest.mark.parametrize("t,heads,d", ROWS)
def test_a_row_without_a_scale_in_mid_sequence(fmt, t, heads, d):
    c = Case(1, t, heads, 2, d, fmt, torch.bfloat16, 16, [900], seed=t + d, spread=0.0)
    clean, lse = c.run(1)
    c.v[0, 411, 0, 3] = torch.inf
    c.fill()
    o, bad = c.run(1)
    assert torch.equal(bad, lse) and torch.equal(o[0, :, heads // 2:], clean[0, :, heads // 2:])
    assert bool(torch.isnan(o[0, :, :heads // 2]).all())
