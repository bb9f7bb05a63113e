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
