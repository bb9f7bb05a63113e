"""The paged cache on the GPU: what is written reads back as its definition
says, bit for bit."""

import math

import pytest
import torch

from draft_helpers import held, quantized
from helpers import assert_same_bits
from voyager_amd import paged

pytestmark = pytest.mark.gpu
FORMATS = ["fp8_e4m3", "int8", None]


def _rows(n, kv, dim, dtype, seed):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(n, 2, kv, dim, generator=g) * torch.exp(2 * torch.randn(n, 2, kv, 1, generator=g))
    return x.to(dtype)


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("n,kv,dim,page", [(1, 1, 64, 16), (8, 8, 128, 16), (37, 2, 256, 48), (5, 3, 8, 1),
                                           (70, 1, 72, 7), (3, 2, 512, 64), (300, 2, 96, 128)])
def test_write_then_read(fmt, dtype, n, kv, dim, page):
    x = _rows(n, kv, dim, dtype, n + dim)
    x[0, 0, 0] = 0.0  # a row of zeros
    x[n // 2, 1, 0, :] = 2.0**-24  # of float16's least, below bfloat16's rounding of nothing
    x[n // 2, 1, 0, 0] = -60000.0  # one large value: the rest of the row is next to nothing
    pages = -(-n // page) + 2
    cache = paged.PagedCache(pages, page, kv, dim, fmt=fmt, dtype=dtype)
    g = torch.Generator().manual_seed(page)
    slots = torch.randperm(pages * page, generator=g)[:n]
    gone = torch.rand(n, generator=g) < 0.2
    slots[gone] = -1 - slots[gone]  # any negative number pads
    xs = x.cuda()
    cache.write(xs[:, 0], xs[:, 1], slots.cuda())
    k, v = cache.read(slots.cuda())
    cache.check()
    for i, (got, name) in enumerate(((k, "k"), (v, "v"))):
        exp = held(x[:, i], fmt).to(dtype)
        exp[gone] = 0
        assert_same_bits(got + 0.0, exp + 0.0, name)  # a zero's sign aside
    if fmt is not None:  # the codes and scales themselves, where the layout says
        codes, scale = quantized(x[:, 0], fmt)
        for j in range(n):
            if gone[j]:
                continue
            s = int(slots[j])
            at = (s // page, slice(None), s % page)
            raw = cache.k[at].cpu()
            got = raw.float() - 128 if fmt == "int8" else raw.view(torch.float8_e4m3fn).float()
            assert torch.equal(got, codes[j]) and torch.equal(cache.k_scale[at].cpu(), scale[j, :, 0])
    # slots that nothing was written to are as they were
    other = torch.tensor(sorted(set(range(pages * page)) - set(slots.tolist())), dtype=torch.int64).cuda()
    assert all(bool((t == 0).all()) for t in cache.read(other))


@pytest.mark.parametrize("fmt", ["fp8_e4m3", "int8"])
def test_rows_that_are_not_finite_read_as_nan(fmt):
    x = _rows(4, 2, 64, torch.bfloat16, 1)
    x[1, 0, 1, 5], x[2, 1, 0, 63], x[3, 0, 0, 0] = math.nan, math.inf, -math.inf
    cache = paged.PagedCache(1, 16, 2, 64, fmt=fmt)
    slots = torch.arange(4).cuda()
    cache.write(x[:, 0].cuda(), x[:, 1].cuda(), slots)
    for i, got in enumerate(cache.read(slots)):
        assert_same_bits(got + 0.0, held(x[:, i], fmt).bfloat16() + 0.0)


@pytest.mark.parametrize("fmt", FORMATS)
def test_views(fmt):
    """A fused projection's rows, rows off 16 bytes, channels not dense, slots with a step."""
    x = _rows(6, 4, 64, torch.bfloat16, 2).cuda()
    slots = torch.arange(6).cuda()
    plain = paged.PagedCache(1, 16, 4, 64, fmt=fmt)
    plain.write(x[:, 0].contiguous(), x[:, 1].contiguous(), slots)
    exp = plain.read(slots)
    odd = torch.empty(6, 4, 71, dtype=torch.bfloat16, device="cuda")[..., 3:67]
    odd.copy_(x[:, 0])
    for k in (x[:, 0], odd, x[:, 0].transpose(1, 2).contiguous().transpose(1, 2),
              x[:, 0].transpose(0, 1).contiguous().transpose(0, 1)):
        c = paged.PagedCache(1, 16, 4, 64, fmt=fmt)
        c.write(k, x[:, 1], torch.arange(0, 12).cuda()[::2] // 2)
        assert all(torch.equal(a, b) for a, b in zip(c.read(torch.arange(12).cuda()[:6]), exp))


def test_slots_past_the_cache_are_left_out_and_told():
    cache = paged.PagedCache(2, 16, 1, 64)
    x = _rows(3, 1, 64, torch.bfloat16, 3).cuda()
    cache.write(x[:, 0], x[:, 1], torch.tensor([32, 5, 1 << 40]).cuda())
    with pytest.raises(RuntimeError, match="outside the cache"):
        cache.check()
    cache.check()  # cleared
    k, _ = cache.read(torch.tensor([5, 33]).cuda())
    assert torch.equal(k[0].cpu(), held(x[1:2, 0].cpu(), "fp8_e4m3").bfloat16()[0]) and bool((k[1] == 0).all())
    with pytest.raises(RuntimeError, match="outside the cache"):
        cache.check()


def test_nothing():
    cache = paged.PagedCache(1, 16, 1, 64)
    none = torch.empty(0, 1, 64, dtype=torch.bfloat16, device="cuda")
    at = torch.empty(0, dtype=torch.int64, device="cuda")
    cache.write(none, none, at)
    assert cache.read(at)[0].shape == (0, 1, 64)


@pytest.mark.parametrize("fmt", FORMATS)
def test_keep_moves_rows_as_they_are(fmt):
    b, t, kv, dim, page = 3, 7, 2, 64, 16
    table = torch.tensor([[5, 0, 3], [2, 7, 1], [8, 4, 6]], dtype=torch.int32)
    context = torch.tensor([13, 0, 40], dtype=torch.int32)  # the tree of the first crosses a page
    cache = paged.PagedCache(9, page, kv, dim, fmt=fmt)
    x = _rows(9 * page, kv, dim, torch.bfloat16, 4).cuda()
    cache.write(x[:, 0], x[:, 1], torch.arange(9 * page).cuda())
    path = torch.tensor([[0, 2, 3, 6, -1, -1, -1], [0, 1, 2, 3, 4, 5, 6], [0, -1, -1, -1, -1, -1, -1]], dtype=torch.int32)
    count = torch.tensor([4, 7, 1], dtype=torch.int32)
    slot = lambda i, p: int(table[i, p // page]) * page + p % page
    exp = list(range(9 * page))
    for i in range(b):
        for j in range(int(count[i])):
            exp[slot(i, int(context[i]) + j)] = slot(i, int(context[i]) + int(path[i, j]))
    was = [y.clone() for y in cache.read(torch.arange(9 * page).cuda())]
    cache.keep(table.cuda(), context.cuda(), path.cuda(), count.cuda())
    cache.check()
    now = cache.read(torch.arange(9 * page).cuda())
    assert all(torch.equal(a, w[torch.tensor(exp).cuda()]) for a, w in zip(now, was))


@pytest.mark.parametrize("path,table,context", [([0, 2, 1], [0, 1], 3), ([0, 5, -1], [0, 1], 3), ([0, 2, -1], [0, 9], 14),
                                                ([0, 2, -1], [0, -1], 14), ([0, 2, -1], [0, 1], 40),
                                                ([0, 2, -1], [0, 1], -3)])
def test_keep_stops_at_what_is_not_there(path, table, context):
    cache = paged.PagedCache(2, 16, 1, 64)
    i = lambda v: torch.tensor(v, dtype=torch.int32).cuda()
    cache.keep(i([table]), i([context]), i([path]), i([3 if path[2] >= 0 else 2]))
    with pytest.raises(RuntimeError, match="not there"):
        cache.check()


def test_captured():
    cache = paged.PagedCache(4, 16, 2, 64, fmt="int8")
    x = _rows(20, 2, 64, torch.bfloat16, 5).cuda()
    slots = torch.arange(20).cuda()

    def step():
        cache.write(x[:, 0], x[:, 1], slots)
        return cache.read(slots)

    step()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step()
    for i in range(3):
        x.mul_(1.37)
        slots.copy_(torch.randperm(64)[:20])
        exp = [held(x[:, j].cpu(), "int8").bfloat16() for j in range(2)]
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(got, exp):
            assert_same_bits(a + 0.0, b + 0.0, f"replay {i}")
