"""Batches whose contexts sum to more keys than 31 bits count, as sequences
that share their pages can."""

import pytest
import torch

from voyager_amd import _lib, paged, speculative

pytestmark = pytest.mark.gpu


def _run(q, cache, table, context, workgroups):
    b, t, heads, d = q.shape
    o, lse = torch.empty_like(q), torch.empty(b, t, heads, dtype=torch.float32, device="cuda")
    sb, st, sh, _ = q.stride()
    desc = bytes(cache.c) + speculative.TREE.pack(
        q.data_ptr(), sb, st, sh, table.data_ptr(), table.stride(0), context.data_ptr(), 0, o.data_ptr(), lse.data_ptr(),
        d ** -0.5, _lib.dtype_code(q.dtype), b, t, heads, table.shape[1], workgroups)
    lib = _lib.load()
    assert lib.vh_tree_attention_workspace_bytes(desc) == 0
    _lib.check(lib.vh_tree_attention(desc, None, 0, _lib.stream_on(q.device)), "vh_tree_attention")
    return o, lse


@pytest.mark.parametrize("nodes", [1, 40])  # a wave's own keys, and shared ones
def test_contexts_of_more_than_31_bits_in_all(nodes):
    """4096 sequences of 524288 positions, all in one page, each one split: as
    the first of them alone."""
    b, ctx, page = 4096, 1 << 19, 16
    if nodes > 1:
        b, ctx = 512, 1 << 22
    g = torch.Generator().manual_seed(1)
    cache = paged.PagedCache(1, page, 1, 64)
    x = torch.randn(2, page, 1, 64, generator=g).bfloat16().cuda()
    cache.write(x[0], x[1], torch.arange(page).cuda())
    table = torch.zeros(1, (ctx + nodes + page - 1) // page, dtype=torch.int32, device="cuda")
    q = torch.randn(1, nodes, 1, 64, generator=g).bfloat16().cuda()
    context = torch.full((b,), ctx, dtype=torch.int32, device="cuda")
    alone = _run(q, cache, table, context[:1], 1)
    every = _run(q.expand(b, nodes, 1, 64).contiguous(), cache, table.expand(b, -1), context, 1)
    cache.check()
    assert bool(torch.isfinite(alone[1]).all())
    for one, all_ in zip(alone, every):
        assert torch.equal(all_, one.expand_as(all_))
