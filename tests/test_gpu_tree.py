"""Attention of a tree of tokens over a paged cache, against float64."""

import math

import pytest
import torch

from draft_helpers import ancestors, attention, attention_tolerance
from voyager_amd import paged, speculative

pytestmark = pytest.mark.gpu
FORMATS = ["fp8_e4m3", "int8", None]


def _parents(b, t, seed):
    g = torch.Generator().manual_seed(seed)
    n = torch.arange(t).expand(b, t)
    return torch.where(n == 0, -1, (torch.rand(b, t, generator=g) * n).long()).int()


def _setup(b, t, heads, kv, d, fmt, dtype, page, contexts, seed=0, spread=1.0):
    """Queries, a filled cache with its pages in any order, and what the cache
    holds, as [b, positions, kv, d] in float64."""
    g = torch.Generator().manual_seed(seed)
    per = -(-(max(contexts) + t) // page) + 1
    pages = b * per + 3
    order = torch.randperm(pages, generator=g)[: b * per]
    table = order.reshape(b, per)
    cache = paged.PagedCache(pages, page, kv, d, fmt=fmt, dtype=dtype)
    x = (torch.randn(2, b, per * page, kv, d, generator=g) * torch.exp(
        spread * torch.randn(2, b, per * page, kv, 1, generator=g))).to(dtype)
    slots = (table[:, :, None] * page + torch.arange(page)).reshape(-1)
    for i in range(b):  # past the tree nothing is written: what lies there is old, not zero
        junk = x[:, i, contexts[i] + t:]
        junk.fill_(math.nan if fmt is None else 7.0)
    flat = x.reshape(2, b * per * page, kv, d).cuda()
    cache.write(flat[0], flat[1], slots.cuda())
    k, v = cache.k.cpu(), cache.v.cpu()
    def rows(codes, scales):
        c = codes.float() if fmt is None else codes.float() - 128 if fmt == "int8" else codes.view(torch.float8_e4m3fn).float()
        c = c.double() if scales is None else c.double() * scales.cpu().double()[..., None]
        return c[table].transpose(2, 3).reshape(b, per * page, kv, d)
    q = torch.randn(b, t, heads, d, generator=g).to(dtype)
    ctx = torch.tensor(contexts, dtype=torch.int32)
    return q, cache, table.int(), ctx, rows(k, cache.k_scale), rows(v, cache.v_scale)


def _compare(got, lse, q, k, v, ctx, see, fmt, scale=None, heads=None):
    d = q.shape[3]
    keys = int(ctx.max()) + q.shape[1]
    ref, rlse, mag, dot = attention(q, k, v, ctx, see, d ** -0.5 if scale is None else scale)
    tol, tlse = attention_tolerance(q.dtype, fmt, d, keys, ref, mag, dot, v[torch.isfinite(v)].abs().max())
    err = (got.cpu().double() - ref).abs()
    assert bool((err <= tol).all()), f"output: {int((err > tol).sum())} beyond, worst {float((err / tol).max()):.2f}"
    empty = torch.isinf(rlse)
    assert torch.equal(torch.isinf(lse.cpu()), empty) and bool((got.cpu()[empty] == 0).all())
    e = (lse.cpu().double() - rlse).abs()[~empty]
    assert bool((e <= tlse[~empty]).all()), f"lse: worst {float((e / tlse[~empty]).max()):.2f}"


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("b,t,heads,kv,d,page,contexts", [
    (1, 1, 4, 1, 128, 16, [0]),            # the first token of a sequence
    (3, 1, 8, 2, 128, 16, [1, 31, 300]),   # single tokens, splits of one step
    (2, 1, 16, 1, 64, 48, [33, 200]),      # 16 rows, pages that end inside a step
    (2, 5, 7, 1, 64, 32, [15, 129]),       # 35 rows: four tiles, the third not full
    (1, 9, 3, 3, 256, 64, [77]),           # a group of one
    (2, 13, 8, 2, 256, 16, [64, 127]),     # two row blocks
    (1, 64, 4, 1, 128, 128, [511]),        # a whole word of nodes, four row blocks
    (2, 70, 2, 1, 64, 16, [5, 90])])       # two words
def test_trees(fmt, dtype, b, t, heads, kv, d, page, contexts):
    q, cache, table, ctx, k, v = _setup(b, t, heads, kv, d, fmt, dtype, page, contexts, seed=t + d)
    parents = _parents(b, t, 5)
    tree = speculative.Tree(parents.cuda())
    o, lse = speculative.tree_attention(q.cuda(), cache, table.cuda(), ctx.cuda(), tree, return_lse=True)
    tree.check()
    cache.check()
    _compare(o, lse, q, k, v, ctx, ancestors(parents), fmt)


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("t,context", [(1, 40), (37, 0), (100, 21)])
def test_without_a_tree_each_sees_those_before(fmt, t, context):
    q, cache, table, ctx, k, v = _setup(2, t, 4, 2, 64, fmt, torch.bfloat16, 16, [context, context // 2], seed=t)
    o, lse = speculative.tree_attention(q.cuda(), cache, table.cuda(), ctx.cuda(), return_lse=True, scale=0.3)
    _compare(o, lse, q, k, v, ctx, torch.ones(2, t, t).tril().bool(), fmt, scale=0.3)
    assert torch.equal(o, speculative.tree_attention(q.cuda(), cache, table.cuda(), ctx.cuda(), scale=0.3))


@pytest.mark.parametrize("fmt", FORMATS)
def test_padding_nodes_see_nothing(fmt):
    q, cache, table, ctx, k, v = _setup(2, 6, 4, 2, 64, fmt, torch.bfloat16, 16, [0, 50], seed=3)
    parents = torch.tensor([[-1, 0, -1, 2, 1, -7], [-1, 0, 1, -1, -1, -1]], dtype=torch.int32)  # 3 is under padding
    o, lse = speculative.tree_attention(q.cuda(), cache, table.cuda(), ctx.cuda(), speculative.Tree(parents.cuda()),
                                        return_lse=True)
    see = ancestors(parents)
    assert not see[0, 2].any() and not see[0, 3].any()
    # a node that pads sees no context either: take its rows out of the reference
    got, rl = o.cpu(), lse.cpu()
    for i in range(2):
        pads = ~see[i].any(-1)
        assert bool((got[i, pads] == 0).all()) and bool((rl[i, pads] == -math.inf).all())
    ref, rlse, mag, dot = attention(q, k, v, ctx, see, 0.125)
    tol, tlse = attention_tolerance(q.dtype, fmt, 64, 56, ref, mag, dot, v[torch.isfinite(v)].abs().max())
    live = see.any(-1)
    assert bool(((got.double() - ref).abs() <= tol)[live].all()) and bool(((rl.double() - rlse).abs() <= tlse)[live].all())


def test_a_bad_parent_is_told():
    parents = torch.tensor([[-1, 0, 2, 1]], dtype=torch.int32)
    tree = speculative.Tree(parents.cuda())
    assert tree.masks[0, :, 0].tolist() == [1, 3, 0, 11]
    with pytest.raises(RuntimeError, match="parent"):
        tree.check()


def test_masks_of_many_nodes():
    parents = _parents(2, 1024, 9)
    parents[1] = torch.arange(-1, 1023)  # a chain
    tree = speculative.Tree(parents.cuda())
    tree.check()
    bits = (tree.masks.cpu()[..., None] >> torch.arange(64)) & 1
    see = bits.reshape(2, 1024, 1024).bool()
    assert torch.equal(see[1], torch.ones(1024, 1024).tril().bool())
    assert torch.equal(see[:1, :, :], ancestors(parents[:1]))


@pytest.mark.parametrize("fmt", FORMATS)
def test_scores_far_apart(fmt):
    """Scores of hundreds, rising along the keys, so that the running maximum
    moves in every step, and value scales over many binades."""
    b, t, d, ctx = 1, 3, 64, 400
    q, cache, table, c, k, v = _setup(b, t, 4, 2, d, fmt, torch.bfloat16, 16, [ctx], seed=8, spread=3.0)
    parents = _parents(b, t, 2)
    o, lse = speculative.tree_attention((q * 8).cuda(), cache, table.cuda(), c.cuda(), speculative.Tree(parents.cuda()),
                                        return_lse=True)
    _compare(o, lse, q * 8, k, v, c, ancestors(parents), fmt)


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("size", [1e-30, 1e20])
def test_small_and_large_queries(fmt, size):
    q, cache, table, c, k, v = _setup(1, 2, 4, 2, 64, fmt, torch.bfloat16, 16, [50], seed=9, spread=0.0)
    q = (q.float() * size).bfloat16()
    scale = 1e-19 if size > 1 else 1.0
    o, lse = speculative.tree_attention(q.cuda(), cache, table.cuda(), c.cuda(), scale=scale, return_lse=True)
    _compare(o, lse, q, k, v, c, torch.ones(1, 2, 2).tril().bool(), fmt, scale=scale)


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("what", [math.nan, math.inf, -math.inf])
def test_what_is_masked_does_not_reach_a_row(fmt, what):
    """Keys and values of one node that are not finite: only rows that see it
    change, and those are not finite."""
    b, t, kv, d, page, ctx = 1, 6, 2, 64, 16, 21
    q, cache, table, c, k, v = _setup(b, t, 4, kv, d, fmt, torch.bfloat16, page, [ctx], seed=10)
    parents = torch.tensor([[-1, 0, 0, 1, 2, 2]], dtype=torch.int32)
    tree = speculative.Tree(parents.cuda())
    args = (cache, table.cuda(), c.cuda(), tree)
    clean, cl = speculative.tree_attention(q.cuda(), *args, return_lse=True)
    pos = ctx + 2
    slot = torch.tensor([int(table[0, pos // page]) * page + pos % page]).cuda()
    kk, vv = cache.read(slot)
    bad = vv.clone()
    bad[0, 0, 5] = what
    cache.write(kk, bad, slot)
    o, lse = speculative.tree_attention(q.cuda(), *args, return_lse=True)
    assert torch.equal(lse, cl)
    sees = ancestors(parents)[0, :, 2]
    head0 = o[0, :, :2].cpu()  # the heads of key head 0
    assert torch.equal(head0[~sees], clean[0, :, :2].cpu()[~sees]) and torch.equal(o[0, :, 2:], clean[0, :, 2:])
    if fmt is None:  # channel by channel
        want = clean[0, :, :2].cpu()[sees].clone()
        want[..., 5] = what
        got = head0[sees]
        assert torch.equal(torch.isnan(got), torch.isnan(want))
        assert bool((got[..., 5] == what).all()) or math.isnan(what)
        rest = torch.arange(d) != 5
        assert torch.equal(got[..., rest], want[..., rest])
    else:
        assert bool(torch.isnan(head0[sees]).all())
    # a key: rows that see it have no finite score sum, the others nothing of it
    bad = kk.clone()
    bad[0, 0, 5] = math.nan
    cache.write(bad, vv, slot)
    o, lse = speculative.tree_attention(q.cuda(), *args, return_lse=True)
    assert torch.equal(lse[0, :, :2].cpu()[~sees], cl[0, :, :2].cpu()[~sees]) and torch.equal(o[0, :, 2:], clean[0, :, 2:])
    assert bool(torch.isnan(lse[0, :, :2].cpu()[sees]).all()) and bool(torch.isnan(o[0, :, :2].cpu()[sees]).all())
    assert torch.equal(o[0, :, :2].cpu()[~sees], clean[0, :, :2].cpu()[~sees])


def test_pages_and_contexts_out_of_range():
    q, cache, table, c, k, v = _setup(3, 2, 4, 2, 64, "int8", torch.bfloat16, 16, [40, 40, 40], seed=11)
    run = lambda tab, ctx: speculative.tree_attention(q.cuda(), cache, tab.cuda(), ctx.cuda(), return_lse=True)
    clean = run(table, c)
    cache.check()
    for page in (-1, cache.pages, 1 << 30):  # keys 16 to 31 of the second sequence are not there
        bad = table.clone()
        bad[1, 1] = page
        o, lse = run(bad, c)
        with pytest.raises(RuntimeError, match="not there"):
            cache.check()
        left = [j for j in range(42) if not 16 <= j < 32]
        see = torch.ones(1, 2, 2).tril().bool()
        _compare(o[1:2], lse[1:2], q[1:2], k[1:2][:, left], v[1:2][:, left], torch.tensor([24]), see, "int8")
        assert all(torch.equal(a[::2], b[::2]) for a, b in zip((o, lse), clean))
    for length in (-1, table.shape[1] * 16 - 1, 1 << 30):
        ctx = c.clone()
        ctx[2] = length
        o, lse = run(table, ctx)
        with pytest.raises(RuntimeError, match="longer than its pages"):
            cache.check()
        assert bool((o[2] == 0).all()) and bool((lse[2] == -math.inf).all())
        assert all(torch.equal(a[:2], b[:2]) for a, b in zip((o, lse), clean))
    # entries past a sequence's last page are not read
    bad = table.clone()
    bad[:, 3:] = -1
    assert all(torch.equal(a, b) for a, b in zip(run(bad, c), clean))
    cache.check()


@pytest.mark.parametrize("fmt", FORMATS)
def test_views_and_streams(fmt):
    q, cache, table, c, k, v = _setup(2, 3, 4, 2, 64, fmt, torch.bfloat16, 16, [40, 9], seed=12)
    exp = speculative.tree_attention(q.cuda(), cache, table.cuda(), c.cuda())
    wide = torch.zeros(2, 3, 9, 64, dtype=q.dtype, device="cuda")
    wide[:, :, 2:6] = q.cuda()
    odd = torch.zeros(2, 3, 4, 67, dtype=q.dtype, device="cuda")
    odd[..., 1:65] = q.cuda()
    long = torch.full((2, table.shape[1] + 5), -1, dtype=torch.int32, device="cuda")
    long[:, : table.shape[1]] = table.cuda()
    for qq in (wide[:, :, 2:6], odd[..., 1:65], q.cuda().transpose(1, 2).contiguous().transpose(1, 2),
               q.cuda().transpose(2, 3).contiguous().transpose(2, 3)):
        assert torch.equal(speculative.tree_attention(qq, cache, long[:, : table.shape[1]], c.cuda()), exp)
    side = torch.cuda.Stream()
    qd, td, cd = q.cuda(), table.cuda(), c.cuda()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = speculative.tree_attention(qd, cache, td, cd)
    side.synchronize()
    assert torch.equal(got, exp)


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("d,t", [(64, 1), (128, 3), (256, 1)])
def test_many_splits(fmt, d, t):
    """A long sequence beside short ones: most splits of the short are empty."""
    contexts = [3000, 0, 130]
    q, cache, table, c, k, v = _setup(3, t, 4, 2, d, fmt, torch.bfloat16, 64, contexts, seed=13)
    o, lse = speculative.tree_attention(q.cuda(), cache, table.cuda(), c.cuda(), return_lse=True)
    _compare(o, lse, q, k, v, c, torch.ones(3, t, t).tril().bool(), fmt)
    again = speculative.tree_attention(q.cuda(), cache, table.cuda(), c.cuda(), return_lse=True)
    assert torch.equal(again[0], o) and torch.equal(again[1], lse)


def test_nothing():
    cache = paged.PagedCache(1, 16, 2, 64)
    i = lambda *s: torch.zeros(*s, dtype=torch.int32, device="cuda")
    for b, t in ((0, 3), (2, 0)):
        q = torch.zeros(b, t, 4, 64, dtype=torch.bfloat16, device="cuda")
        assert speculative.tree_attention(q, cache, i(b, 1), i(b)).shape == q.shape


def test_captured():
    q, cache, table, c, k, v = _setup(2, 4, 4, 2, 64, "fp8_e4m3", torch.bfloat16, 16, [200, 30], seed=14)
    q, table, c, parents = q.cuda(), table.cuda(), c.cuda(), _parents(2, 4, 1).cuda()
    run = lambda: speculative.tree_attention(q, cache, table, c, speculative.Tree(parents), return_lse=True)
    run()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = run()
    for i in range(3):
        q.mul_(-1.1)
        c.copy_(torch.tensor([150 + 20 * i, 3 * i], dtype=torch.int32))
        parents.copy_(_parents(2, 4, 20 + i))
        exp = run()
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, exp)), f"replay {i}"


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("t", [2, 20])
def test_pages_past_32_bits(fmt, t):
    """The last pages of a cache whose keys alone are over 4 GiB: written,
    attended to, moved and read as those of a small one are."""
    kv, d, page, per = 8, 256, 64, 4
    b = 2
    count = (1 << 32) // (kv * d * page * (1 if fmt else 2)) + 16
    g = torch.Generator().manual_seed(15)
    x = torch.randn(2, b * per * page, kv, d, generator=g).bfloat16().cuda()
    q = torch.randn(b, t, 16, d, generator=g).bfloat16().cuda()
    context = torch.tensor([per * page - t, 77], dtype=torch.int32).cuda()
    tree = speculative.Tree(_parents(b, t, 5).cuda())
    kept = torch.full((b, t), -1, dtype=torch.int32)
    kept[:, 0], kept[:, 1] = 0, t - 1
    results = []
    for pages in (b * per, count):
        cache = paged.PagedCache(pages, page, kv, d, fmt=fmt)
        table = (pages - 1 - torch.arange(b * per)).reshape(b, per)
        slots = (table[:, :, None] * page + torch.arange(page)).flatten().cuda()
        table = table.int().cuda()
        cache.write(x[0], x[1], slots)
        o, lse = speculative.tree_attention(q, cache, table, context, tree, return_lse=True)
        cache.keep(table, context, kept.cuda(), torch.full((b,), 2, dtype=torch.int32, device="cuda"))
        results.append((o, lse, *cache.read(slots)))
        cache.check()
    assert all(torch.equal(near, far) for near, far in zip(*results))
