"""Scores of a part of a batch's logits on the GPU: rows in place."""

import pytest
import torch

from voyager_amd import score

pytestmark = pytest.mark.gpu


def _batch(shape, dtype=torch.bfloat16, seed=0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return (torch.randn(*shape, generator=g, device="cuda") * 3).to(dtype)


VIEWS = {
    "all but a sequence's last": lambda x: x[:, :-1],
    "all but its first": lambda x: x[:, 1:],
    "every other one": lambda x: x[:, ::2],
    "some sequences": lambda x: x[1:, 2:5],
    "one of each sequence": lambda x: x[:, 3],
    "sequences inside": lambda x: x.transpose(0, 1)[:-1],
    "part of the vocabulary": lambda x: x[:, :-1, 5:-7],
    "one sequence for all": lambda x: x[:1, :-1].expand(3, -1, -1),
    "one row for all": lambda x: x[:1, :1].expand(3, 6, -1),
    "a batch of batches": lambda x: x[:, None, :-1],
    "nothing of each": lambda x: x[:, :0],
}


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("vocab,top", [(1000, 3), (40000, 0), (40000, 5)])
@pytest.mark.parametrize("view", VIEWS)
def test_views_are_as_their_copies(dtype, vocab, top, view):
    part = VIEWS[view](_batch((3, 9, vocab), dtype))
    tokens = torch.randint(-1, part.shape[-1], part.shape[:-1], generator=torch.Generator().manual_seed(1)).cuda()

    def run(x):
        x = x.detach().requires_grad_()
        s = score.token_scores(x, tokens, top=top)
        out = [y for y in s if y is not None]
        ends = [y for y in out if y.is_floating_point()]
        g = torch.Generator().manual_seed(2)
        (dx,) = torch.autograd.grad(ends, x, [torch.randn(y.shape, generator=g).cuda() for y in ends])
        return [y.detach() for y in out] + [dx]

    for a, b in zip(run(part), run(part.contiguous())):
        assert a.shape == b.shape and torch.equal(a.nan_to_num(7), b.nan_to_num(7))


@pytest.mark.parametrize("view", ["all but a sequence's last", "one sequence for all", "sequences inside", "every other one"])
def test_views_are_not_copied(view):
    """A call allocates its results, not the logits again; its gradient the gradient alone."""
    x = _batch((4, 129, 32000))
    part = VIEWS[view](x).detach()
    tokens = torch.zeros(part.shape[:-1], dtype=torch.int64, device="cuda")
    size = part.numel() * part.element_size()

    def most(f):
        torch.cuda.synchronize()
        torch.cuda.reset_peak_memory_stats()
        before = torch.cuda.memory_allocated()
        y = f()
        return torch.cuda.max_memory_allocated() - before, y

    used, _ = most(lambda: score.token_scores(part, tokens, top=3))
    assert used < size // 4
    s = score.token_scores(part.requires_grad_(), tokens)
    ones = torch.ones_like(s.logprob)
    used, (dx,) = most(lambda: torch.autograd.grad(s.logprob, part, ones))
    assert used < size + size // 4


def test_entries_of_rows_at_one_distance():
    """The C entries without batches, beside the call."""
    from voyager_amd import _lib

    x = _batch((6, 5003), torch.float16)
    tokens = torch.tensor([0, 5002, -1, 7, 5003, 9]).cuda()
    leaf = x.clone().requires_grad_()
    want = score.token_scores(leaf, tokens, top=2)
    g = torch.randn(6, generator=torch.Generator().manual_seed(3)).cuda()
    (grad,) = torch.autograd.grad(want.logprob, leaf, g)
    f = lambda *s: torch.empty(*s, device="cuda")
    logprob, entropy, stats, best, out = f(6), f(6), f(6, 2), f(6, 2), torch.empty_like(x)
    index = torch.empty(6, 2, dtype=torch.int64, device="cuda")
    lib, stream = _lib.load(), _lib.stream_on(x.device)

    def desc(gp):
        return score.SCORE.pack(x.data_ptr(), 5003, tokens.data_ptr(), 6, 5003, logprob.data_ptr(), entropy.data_ptr(),
                                stats.data_ptr(), best.data_ptr(), index.data_ptr(), gp, 0, 0, out.data_ptr(),
                                _lib.dtype_code(x.dtype), 2)

    need = lib.vh_score_workspace_bytes(desc(0))
    work = torch.empty(max(need, 1), dtype=torch.uint8, device="cuda")
    assert lib.vh_score(desc(0), work.data_ptr(), need, stream) == 0
    assert lib.vh_score_backward(desc(g.data_ptr()), stream) == 0
    for a, b in ((logprob, want.logprob), (entropy, want.entropy), (best, want.top_logprob), (index, want.top_token), (out, grad)):
        assert torch.equal(a.nan_to_num(7), b.detach().nan_to_num(7))
