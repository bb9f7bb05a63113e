"""A captured training step's gradients, each beside its own size, and scores
that are NaN exactly where the definition's are."""

import math
import os
import sys

import pytest
import torch

from pass_helpers import scores
from voyager_amd import score

pytestmark = pytest.mark.gpu
sys.path.insert(0, os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "examples"))


def _documents(lengths):
    g = torch.Generator().manual_seed(1)
    return [torch.randint(0, 512, (n,), generator=g).tolist() for n in lengths]


def test_gradients_of_a_captured_step():
    """Replays on other documents, from the same weights, against the step by
    itself.  The same kernels in the same order, but for the embedding's gradient,
    which is added up in bfloat16 in any order: at most 300 rows of 512 tokens,
    of which one comes 6 times at most: under 2^-6 of its norm."""
    import packed_training as example
    from voyager_amd import prompt

    batches = [example.pack(_documents(n), 300) for n in ((100, 50, 150), (3, 200, 40), (1, 1, 290))]
    assert max(int(torch.bincount(b[0][b[1] >= 0]).max()) for b in batches) <= 6
    weights = torch.ones(300, device="cuda")
    model, held = example.Model(layers=2), [t.clone() for t in batches[0]]

    def step(tokens, targets, positions, offsets):
        loss = example.loss_of(model, tokens, targets, positions, prompt.Packing(offsets, 300), weights, entropy=0.3)
        return torch.autograd.grad(loss, model.parameters())

    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        step(*held)
    torch.cuda.current_stream().wait_stream(s)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step(*held)
    for batch in (*batches, batches[0]):
        for t, new in zip(held, batch):
            t.copy_(new)
        for y in got:
            y.zero_()
        graph.replay()
        torch.cuda.synchronize()
        for y, r in zip(got, step(*batch)):
            size = float(r.double().norm())
            assert size > 0 and float((y.double() - r.double()).norm()) <= 2.0**-6 * size


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("vocab", [700, 40000])
def test_nan_where_the_definition_has_it(dtype, vocab):
    g = torch.Generator().manual_seed(vocab)
    x = (torch.randn(7, vocab, generator=g) * 3).to(dtype).cuda()
    x[0, 5] = math.nan
    x[1] = -math.inf
    x[2, 100:] = -math.inf
    x[6] = torch.finfo(dtype).min
    tokens = torch.tensor([1, 2, 300, vocab, 4, -1, 0]).cuda()
    gs = [torch.randn(7, generator=g).cuda(), torch.randn(7, generator=g).cuda(), torch.randn(7, 3, generator=g).cuda()]
    want = scores(x, tokens, 3, *gs)
    leaf = x.clone().requires_grad_()
    got = score.token_scores(leaf, tokens, top=3)
    (dx,) = torch.autograd.grad([got.logprob, got.entropy, got.top_logprob], leaf, gs)
    for y, r, name in zip([*got, dx], want, ("logprob", "entropy", "alternatives", "tokens", "gradient")):
        if name == "tokens":
            assert torch.equal(y, r)
            continue
        assert torch.equal(torch.isnan(y), torch.isnan(r)), name
        assert torch.equal(torch.isinf(y), torch.isinf(r)), name
