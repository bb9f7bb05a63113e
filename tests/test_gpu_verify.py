"""The choice among drafted tokens on the GPU against the definition, read one
node at a time in float64 on the CPU: equal, number for number."""

import pytest
import torch

from draft_helpers import verify as plain
from voyager_amd import speculative

pytestmark = pytest.mark.gpu


def _parents(b, t, seed, chain=False):
    n = torch.arange(t).expand(b, t)
    if chain:
        return (n - 1).int()
    g = torch.Generator().manual_seed(seed)
    return torch.where(n == 0, -1, (torch.rand(b, t, generator=g).pow(1.5) * n).long()).int()


def _probabilities(b, t, vocab, seed, near=0.5):
    g = torch.Generator().manual_seed(seed)
    z = torch.randn(b, t, vocab, generator=g) * 2
    return z.softmax(-1), (z + near * torch.randn(b, t, vocab, generator=g)).softmax(-1)


def _run(target, parents, tokens, u, r, draft=None):
    tree = speculative.Tree(parents.cuda())
    got = speculative.verify(target.cuda(), tokens.cuda(), tree, u.cuda(), r.cuda(), None if draft is None else draft.cuda())
    assert [x.dtype for x in got] == [torch.int64, torch.int32, torch.int32]
    return [x.cpu().tolist() for x in got]


def _inputs(b, t, vocab, seed):
    g = torch.Generator().manual_seed(seed)
    return torch.rand(b, t, generator=g), torch.rand(b, generator=g)


@pytest.mark.parametrize("b,t,vocab", [(1, 1, 1), (3, 1, 7), (4, 6, 50), (16, 6, 4097), (2, 64, 9000), (5, 33, 12001),
                                       (2, 1000, 300)])
@pytest.mark.parametrize("chain", [False, True])
def test_chosen(b, t, vocab, chain):
    """A node's children are its best tokens, some of them twice."""
    target, draft = _probabilities(b, t, vocab, t + vocab)
    parents = _parents(b, t, 3, chain)
    above = parents.clamp(min=0).long()
    g = torch.Generator().manual_seed(7)
    best = draft.topk(min(vocab, 6), -1).indices
    pick = torch.randint(0, best.shape[-1], (b, t), generator=g)
    tokens = best[torch.arange(b)[:, None], above, pick]
    for seed in range(3):
        u, r = _inputs(b, t, vocab, seed)
        u = u * (0.2, 1.0, 0.6)[seed]
        assert _run(target, parents, tokens, u, r) == [*plain(target, parents, tokens, u, r)]


@pytest.mark.parametrize("b,t,vocab", [(1, 6, 32), (8, 6, 4096), (3, 12, 5000), (2, 40, 777)])
@pytest.mark.parametrize("chain", [False, True])
def test_sampled(b, t, vocab, chain):
    """Children sampled from the draft, several of a node: what a rejected one
    leaves is summed before the next is tried."""
    target, draft = _probabilities(b, t, vocab, t + vocab, near=1.0)
    parents = _parents(b, t, 4, chain)
    g = torch.Generator().manual_seed(8)
    above = parents.clamp(min=0).long()
    rows = draft.gather(1, above[:, :, None].expand(b, t, vocab)).reshape(b * t, vocab)
    tokens = torch.multinomial(rows, 1, generator=g).reshape(b, t)
    for seed in range(3):
        u, r = _inputs(b, t, vocab, seed)
        assert _run(target, parents, tokens, u, r, draft) == [*plain(target, parents, tokens, u, r, draft)]


def test_draft_equal_to_the_target_leaves_nothing():
    """The rest is nothing after a rejection (u = 1 cannot be drawn, but a
    token of no probability can be drafted): it is left as it was."""
    target, _ = _probabilities(4, 3, 64, 1)
    target[..., 5] = 0
    parents = torch.tensor([[-1, 0, 0]] * 4, dtype=torch.int32)
    tokens = torch.full((4, 3), 5)
    u, r = _inputs(4, 3, 64, 2)
    got = _run(target, parents, tokens, u, r, target)
    assert got == [*plain(target, parents, tokens, u, r, target)] and got[2] == [1] * 4


def test_tokens_outside_the_vocabulary_are_never_taken():
    target, draft = _probabilities(2, 5, 40, 3)
    parents = _parents(2, 5, 5)
    tokens = torch.tensor([[0, -1, 40, 1 << 40, 3], [0, 40, -5, 39, -(1 << 40)]])
    u, r = torch.zeros(2, 5), torch.tensor([0.0, 0.9999])
    for d in (None, draft):
        assert _run(target, parents, tokens, u, r, d) == [*plain(target, parents, tokens, u, r, d)]


def test_padding_nodes_are_never_taken():
    target, _ = _probabilities(1, 5, 40, 4)
    parents = torch.tensor([[-1, -1, 0, 1, 7]], dtype=torch.int32)
    tokens = torch.tensor([[0, 1, 2, 3, 4]])
    u, r = torch.zeros(1, 5), torch.tensor([0.5])
    got = _run(target, parents, tokens, u, r)
    assert got[1][0][:2] == [0, 2] and got[2] == [2]


@pytest.mark.parametrize("r", [0.0, 2.0**-24, 0.5, 1 - 2.0**-24])
def test_ends_of_the_range(r):
    """Probabilities with zeros at both ends and in between, in exact sums."""
    vocab = 8200
    target = torch.zeros(1, 1, vocab)
    target[0, 0, 17] = 0.25
    target[0, 0, 4095:4097] = 0.125
    target[0, 0, 8190] = 0.5
    u = torch.zeros(1, 1)
    rr = torch.tensor([r])
    tokens, parents = torch.zeros(1, 1, dtype=torch.int64), torch.tensor([[-1]], dtype=torch.int32)
    got = _run(target, parents, tokens, u, rr)
    assert got == [*plain(target, parents, tokens, u, rr)] and float(target[0, 0, got[0][0][0]]) > 0


def test_no_distribution():
    vocab = 100
    tokens, parents = torch.zeros(2, 1, dtype=torch.int64), torch.tensor([[-1]] * 2, dtype=torch.int32)
    target = torch.zeros(2, 1, vocab)
    target[1, 0, 50] = float("nan")
    told, path, count = _run(target, parents, tokens, torch.zeros(2, 1), torch.tensor([0.3, 0.3]))
    assert told == [[vocab - 1], [0]] and count == [1, 1]


def test_views():
    target, draft = _probabilities(3, 4, 60, 6)
    parents = _parents(3, 4, 0, chain=True)
    tokens = draft.argmax(-1).roll(1, 1)
    u, r = _inputs(3, 4, 60, 1)
    exp = _run(target, parents, tokens, u, r, draft)
    wide = torch.zeros(3, 4, 2, 61, device="cuda")
    wide[:, :, 1, 1:] = target.cuda()
    tree = speculative.Tree(parents.cuda().t().contiguous().t())
    back = draft.cuda().transpose(1, 2).contiguous().transpose(1, 2)
    got = speculative.verify(wide[:, :, 1, 1:], tokens.cuda().t().contiguous().t(), tree, u.cuda(), r.cuda(), back)
    assert [x.cpu().tolist() for x in got] == exp


def test_refusals():
    target, draft = (x.cuda() for x in _probabilities(2, 3, 10, 1))
    tree = speculative.Tree(_parents(2, 3, 1).cuda())
    tokens, (u, r) = torch.zeros(2, 3, dtype=torch.int64).cuda(), (x.cuda() for x in _inputs(2, 3, 10, 1))
    ok = dict(target=target, tokens=tokens, tree=tree, u=u, r=r, draft=draft)
    speculative.verify(**ok)
    for bad in (dict(target=target.double()), dict(target=target[:, :2]), dict(target=target[0]),
                dict(target=target[..., :0], draft=None), dict(draft=draft[..., :9]), dict(tokens=tokens.int()),
                dict(tokens=tokens[:1]), dict(u=u.double()), dict(u=u[:, :2]), dict(r=r[:1]), dict(r=r.cpu())):
        with pytest.raises(ValueError, match="verify"):
            speculative.verify(**{**ok, **bad})


@pytest.mark.parametrize("sampled", [False, True])
def test_captured(sampled):
    b, t, vocab = 3, 6, 5000
    target, draft = (x.cuda() for x in _probabilities(b, t, vocab, 9))
    parents = _parents(b, t, 0, chain=True).cuda()
    tokens = draft.argmax(-1).roll(1, 1)
    u, r = (x.cuda() for x in _inputs(b, t, vocab, 1))
    tree = speculative.Tree(parents)
    run = lambda: speculative.verify(target, tokens, tree, u, r, draft if sampled else None)
    run()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = run()
    for i in range(3):
        u.copy_(torch.rand(b, t))
        r.copy_(torch.rand(b))
        exp = run()
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, exp)), f"replay {i}"
