"""Scores of batches of rows without a GPU: the C entries' refusals, which come
before a launch, the descriptor, and how a tensor's rows are told."""

import pytest
import torch

from test_pass_host import P, _size
from voyager_amd import _lib, score


def _batched(entry="vh_score_batched", work=P, work_bytes=1 << 40, batch_rows=2, batch_st=5000, **kw):
    a = dict(logits=P, logits_st=1000, tokens=P, rows=4, vocab=1000, logprob=P, entropy=P, stats=P, top_logprob=P, top_token=P,
             g_logprob=P, g_entropy=0, g_top=0, grad=P, dtype=_lib.VH_F32, top=3)
    a.update(kw)
    d, lib = score.SCORE.pack(*a.values()) + score.BATCHED.pack(batch_rows, batch_st), _lib.load()
    if entry == "vh_score_batched":
        return lib.vh_score_batched(d, work, work_bytes, None)
    return lib.vh_score_batched_backward(d, None)


def test_descriptor_is_as_long_as_the_header_says():
    assert _size("vh_score_batched_desc") == score.SCORE.size + score.BATCHED.size


@pytest.mark.parametrize("entry", ["vh_score_batched", "vh_score_batched_backward"])
@pytest.mark.parametrize("kw", [dict(batch_rows=0), dict(batch_rows=-2), dict(dtype=_lib.VH_U8), dict(rows=-1), dict(rows=1 << 23),
                                dict(vocab=0), dict(top=65), dict(logits=0), dict(tokens=0), dict(entropy=0),
                                dict(rows=1 << 22, vocab=1 << 17)])
def test_entries_refuse(entry, kw):
    assert _batched(entry, **kw) == 1 and _lib.load().vh_last_error().startswith(entry.encode() + b":")


def test_entries_need_their_tensors_and_nothing_for_no_rows():
    for kw in (dict(logprob=0), dict(top_token=0), dict(vocab=100000, work=None), dict(vocab=100000, work_bytes=8)):
        assert _batched(**kw) == 1
    for kw in (dict(stats=0), dict(grad=0)):
        assert _batched("vh_score_batched_backward", **kw) == 1
    assert _batched(rows=0, work=None, work_bytes=0) == 0 and _batched("vh_score_batched_backward", rows=0) == 0


@pytest.mark.parametrize("view", [
    lambda x: x, lambda x: x[:, :-1], lambda x: x[:, 1:], lambda x: x[:, ::2], lambda x: x[:, 2], lambda x: x[1], lambda x: x[1, 2],
    lambda x: x.transpose(0, 1), lambda x: x.transpose(0, 1)[:3], lambda x: x[:, :, 2:5], lambda x: x[:1, :-1].expand(4, -1, -1),
    lambda x: x[:1, :1].expand(2, 3, -1), lambda x: x[:, None, 1:], lambda x: x.view(2, 2, 5, 7)[:, :, :-1],
    lambda x: x.view(2, 2, 5, 7)[:, 1:, :-1], lambda x: x[:, :, ::2], lambda x: x.transpose(1, 2), lambda x: x[:, :, 3:4],
    lambda x: x[:, :0], lambda x: x.view(2, 2, 5, 7).transpose(0, 2)])
def test_rows_are_where_they_are_told_to_be(view):
    x = torch.arange(4 * 5 * 7).float().view(4, 5, 7)
    v = view(x)
    held, step, batch_rows, batch_step = score._rows(v)
    want = v.reshape(-1, v.shape[-1]) if v.numel() else v.new_zeros(0, v.shape[-1])
    memory = torch.as_strided(held, (held.untyped_storage().size() // 4,), (1,), 0)
    for i, row in enumerate(want):
        at = held.storage_offset() + i // batch_rows * batch_step + i % batch_rows * step
        assert torch.equal(memory[at:at + v.shape[-1]], row)
