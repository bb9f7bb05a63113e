"""The choice among drafted tokens where nothing is left, or no number: the
token told is one that the target can give."""

import pytest
import torch

from voyager_amd import speculative

pytestmark = pytest.mark.gpu


def _run(target, parents, tokens, u, r, draft=None):
    tree = speculative.Tree(torch.tensor(parents, dtype=torch.int32).cuda())
    tensors = (torch.as_tensor(x).cuda() for x in (target, tokens))
    got = speculative.verify(*tensors, tree, torch.tensor(u).cuda(), torch.tensor(r).cuda(),
                             None if draft is None else draft.cuda())
    return [x.cpu().tolist() for x in got]


@pytest.mark.parametrize("vocab", [10, 5000])
@pytest.mark.parametrize("r", [0.0, 0.5, 1 - 2.0**-24])
def test_children_that_cover_the_target(vocab, r):
    """Two tokens share a target whose float32 probabilities sum to a little
    under 1, and u is the largest number there is: both children are rejected,
    and the one taken out last is put back."""
    target = torch.zeros(6, 5, vocab)
    target[:, 0, 2], target[:, 0, 6] = 0.3, 0.7 - 2.0**-22
    tokens = torch.tensor([[0, 2, 6, 0, 0], [0, 6, 2, 0, 0],  # each order; the rest pad
                           [0, 2, 6, 2, 0],                   # one of them once more
                           [0, 2, 6, 3, vocab],               # then one of no probability, and one outside
                           [0, 2, 6, -1, 1 << 40],
                           [0, 6, 6, 6, 6]])                  # one of the two alone: the other is left
    parents = [[-1, 0, 0, -1, -1]] * 2 + [[-1, 0, 0, 0, -1]] + [[-1, 0, 0, 0, 0]] * 3
    u = [[1 - 2.0**-24] * 5] * 6
    told, path, count = _run(target, parents, tokens, u, [r] * 6)
    # 6, then 2: mass is 1 - 0.7 + 2^-22, more than 2 has
    assert [t[0] for t in told] == [6, 2, 6, 6, 6, 2]
    assert count == [1] * 6 and all(p == [0, -1, -1, -1, -1] for p in path) and all(t[1:] == [-1] * 4 for t in told)


def test_children_that_cover_it_deeper_in_the_tree():
    """The same at the end of a path, among children of other nodes."""
    vocab = 5000
    target = torch.zeros(1, 6, vocab)
    target[0, 0, 4500] = 1.0
    target[0, 2, 4999], target[0, 2, 1] = 0.5, 0.5 - 2.0**-23
    tokens = torch.tensor([[0, 4000, 4500, 4999, 1, 1]])
    told, path, count = _run(target, [[-1, 0, 0, 2, 2, 1]], tokens, [[1 - 2.0**-24] * 6], [0.2])
    assert told == [[4500, 1, -1, -1, -1, -1]] and path == [[0, 2, -1, -1, -1, -1]] and count == [2]


def test_many_children_that_cover_it():
    vocab = n = 1000
    target = torch.full((1, n, vocab), 2.0**-10)  # 0.976 in all
    tokens = torch.arange(-1, n - 1)[None].clamp(min=0)
    target[0, :, 999] = 0.0
    told, _, count = _run(target, [[-1] + [0] * (n - 1)], tokens, [[1 - 2.0**-24] * n], [0.9])
    assert told[0][0] == 998 and count == [1]


@pytest.mark.parametrize("vocab", [40, 5000])
@pytest.mark.parametrize("rejected", [0, 1, 2])
def test_a_row_that_holds_a_nan_tells_its_start(vocab, rejected):
    """With none, one or two sampled children rejected before."""
    g = torch.Generator().manual_seed(vocab)
    draft = torch.randn(1, 3, vocab, generator=g).softmax(-1)
    target = torch.randn(1, 3, vocab, generator=g).softmax(-1)
    target[0, 0, 7], target[0, 0, 8] = 0.0, 0.0
    target[0, 0, vocab - 5] = float("nan")
    parents = [[-1] + [0] * rejected + [-1] * (2 - rejected)]
    told, path, count = _run(target, parents, torch.tensor([[0, 7, 8]]), [[0.5] * 3], [0.4], draft)
    assert told == [[0, -1, -1]] and path == [[0, -1, -1]] and count == [1]
