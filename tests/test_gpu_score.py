"""Scores of given tokens on the GPU, and their gradients, against float64."""

import math

import pytest
import torch

from pass_helpers import score_tolerances, scores, within
from voyager_amd import score

pytestmark = pytest.mark.gpu
DTYPES = [torch.bfloat16, torch.float16, torch.float32]


def _logits(rows, vocab, dtype, seed=0, spread=3.0):
    g = torch.Generator().manual_seed(seed + rows + vocab)
    return (torch.randn(rows, vocab, generator=g) * spread).to(dtype).cuda()


def _tokens(rows, vocab, seed=0):
    return torch.randint(0, vocab, (rows,), generator=torch.Generator().manual_seed(seed)).cuda()


def check(logits, tokens, top, grads=True, seed=0):
    x = logits.detach().clone().as_strided(logits.shape, logits.stride()) if logits.is_contiguous() else logits.detach()
    x = x.requires_grad_(grads)
    got = score.token_scores(x, tokens, top=top)
    rows, vocab = logits.shape
    g = torch.Generator().manual_seed(seed)
    gs = [torch.randn(rows, generator=g).cuda(), torch.randn(rows, generator=g).cuda(), torch.randn(rows, top, generator=g).cuda()]
    ref = scores(logits.detach(), tokens, top, *gs)
    tol = score_tolerances(logits.detach(), ref, *gs)
    for y, r, e, what in zip(got[:2], ref[:2], tol[:2], ("logprob", "entropy")):
        same = torch.isinf(r) & (y.double() == r)
        within(torch.where(same, 0.0, y.double()), torch.where(same, 0.0, r), e, what)
    if top:
        assert torch.equal(got.top_token, ref[3])
        same = torch.isinf(ref[2]) & (got.top_logprob.double() == ref[2])
        within(torch.where(same, 0.0, got.top_logprob.double()), torch.where(same, 0.0, ref[2]), tol[2], "alternatives")
    else:
        assert got.top_logprob is None and got.top_token is None
    if grads:
        ends = [got.logprob, got.entropy] + ([got.top_logprob] if top else [])
        (dx,) = torch.autograd.grad(ends, x, gs[:len(ends)])
        assert dx.dtype == x.dtype and dx.shape == x.shape
        within(dx, ref[4], tol[3], "gradient")
    return got


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,vocab,top", [
    (1, 1, 1), (1, 1, 0), (3, 2, 2), (5, 7, 3), (2, 64, 64), (4, 1000, 5), (1, 4095, 20), (1, 4097, 64), (2, 32000, 5),
    (1, 128000, 20), (300, 509, 1), (2, 50257, 64), (257, 8193, 2), (1, 262144, 7)])
def test_values_and_gradients(dtype, rows, vocab, top):
    check(_logits(rows, vocab, dtype), _tokens(rows, vocab), top)


def test_the_most_rows():
    """The last rows, beside a call of their own."""
    rows = (1 << 23) - 1
    g = torch.Generator(device="cuda").manual_seed(7)
    x = torch.randn(rows, 3, generator=g, device="cuda", dtype=torch.float16)
    t = torch.randint(-1, 3, (rows,), generator=g, device="cuda")

    def run(x, t):
        x = x.detach().requires_grad_()
        s = score.token_scores(x, t, top=2)
        return [*(y.detach() for y in s), *torch.autograd.grad((s.logprob + s.entropy).sum(), x)]
    for some in (slice(0, 1000), slice(-1000, None)):
        for y, z in zip(run(x, t), run(x[some], t[some])):
            assert torch.equal(y[some], z)


def test_the_largest_vocabulary():
    check(_logits(1, 1 << 20, torch.float32), _tokens(1, 1 << 20), 64)
    check(_logits(2, (1 << 20) - 3, torch.bfloat16), _tokens(2, 1000), 3)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("vocab", [1000, 40000])
def test_ties_go_to_the_lowest_index(dtype, vocab):
    """Rows of one value, of few values, and rising ones, where every entry is the largest so far."""
    flat = torch.full((1, vocab), 1.5)
    few = torch.randint(0, 3, (1, vocab), generator=torch.Generator().manual_seed(1)).float()
    last = torch.zeros(1, vocab)
    last[0, -30:] = 1.0
    signs = torch.zeros(1, vocab)
    signs[0, ::2] = -0.0
    rising = torch.arange(vocab).float()[None] / vocab
    x = torch.cat((flat, few, last, signs, rising, -rising)).to(dtype).cuda()
    for top in (1, 20, 64):
        check(x, _tokens(6, vocab), top)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("vocab", [999, 40000])
def test_masked_vocabularies(dtype, vocab):
    """Entries of -inf and of the type's lowest value; rows with fewer finite entries than alternatives."""
    x = _logits(6, vocab, dtype)
    x[0, 1:] = -math.inf
    x[1, : vocab - 3] = -math.inf
    x[2, torch.arange(vocab) % 100 != 7] = -math.inf
    x[3, torch.arange(vocab) % 100 != 7] = torch.finfo(dtype).min
    x[4, 0] = -math.inf
    tokens = torch.tensor([0, vocab - 1, 7, 7, 0, 3]).cuda()
    check(x, tokens, 0)
    for top in (2, 64):
        check(x, tokens, top)


@pytest.mark.parametrize("dtype", DTYPES)
def test_far_values(dtype):
    x = _logits(3, 5000, dtype)
    most = torch.finfo(dtype).max
    x[0, 17] = most
    x[1] = -most
    x[2] *= 100 if dtype == torch.float16 else 1e4
    got = check(x, torch.tensor([17, 5, 9]).cuda(), 4, grads=False)
    assert float(got.logprob[0]) == 0 and abs(float(got.logprob[1]) + math.log(5000)) < 1e-5


@pytest.mark.parametrize("vocab", [700, 70000])
def test_rows_without_probabilities_stay_their_own(vocab):
    x = _logits(6, vocab, torch.bfloat16)
    tokens = _tokens(6, vocab)
    good = score.token_scores(x, tokens, top=3)
    bad = x.clone()
    bad[0, 5] = math.nan
    bad[1, 6] = math.inf
    bad[2] = -math.inf
    bad[3, 7] = -math.nan
    bad.requires_grad_()
    got = score.token_scores(bad, tokens, top=3)
    for y, z in zip(got, good):
        assert torch.equal(y[4:], z[4:])
        if y.is_floating_point():
            assert bool(torch.isnan(y[:4]).all())
    assert got.top_token[0, 0] == 5 and got.top_token[1, 0] == 6 and got.top_token[2].tolist() == [0, 1, 2] and got.top_token[3, 0] == 7
    (dx,) = torch.autograd.grad(got.logprob.nan_to_num(0).sum() + got.logprob.sum(), bad)
    assert bool(torch.isfinite(dx[4:]).all()) and bool(torch.isnan(dx[:4]).all())


@pytest.mark.parametrize("vocab", [600, 66000])
def test_padding_and_tokens_past_the_vocabulary(vocab):
    x = _logits(5, vocab, torch.float32)
    tokens = torch.tensor([-1, 3, vocab, -100, vocab - 1]).cuda()
    x[3] = math.nan  # a row that pads is not read
    check(x.nan_to_num(0.5), tokens, 4)
    x.requires_grad_()
    got = score.token_scores(x, tokens, top=4)
    assert got.logprob[[0, 3]].tolist() == [0, 0] and got.top_token[0].tolist() == [-1] * 4 and bool(torch.isnan(got.logprob[2]))
    (dx,) = torch.autograd.grad(got.logprob.sum() + got.entropy.sum() + got.top_logprob.sum(), x)
    assert not bool(dx[0].any()) and not bool(dx[3].any()) and bool(torch.isnan(dx[2]).all()) and bool(torch.isfinite(dx[1]).all())


def test_some_gradients_only():
    x = _logits(3, 3000, torch.float32).requires_grad_()
    tokens, z = _tokens(3, 3000), torch.zeros(3).cuda()
    g = torch.randn(3, generator=torch.Generator().manual_seed(1)).cuda()
    t = torch.randn(3, 5, generator=torch.Generator().manual_seed(2)).cuda()
    for which in range(3):
        got = score.token_scores(x, tokens, top=5)
        given = [g if which == 0 else z, g if which == 1 else z, t if which == 2 else torch.zeros_like(t)]
        ref = scores(x.detach(), tokens, 5, *given)
        (dx,) = torch.autograd.grad(got[which], x, given[which])
        within(dx, ref[4], score_tolerances(x.detach(), ref, *given)[3], f"gradient of output {which}")


def test_no_second_gradient():
    x = _logits(3, 100, torch.float32).requires_grad_()
    with pytest.raises(RuntimeError, match="differentiable once"):
        torch.autograd.grad(score.token_scores(x, _tokens(3, 100)).logprob.sum(), x, create_graph=True)


def test_the_token_among_the_alternatives():
    """The same entry twice: both gradients are added."""
    x = _logits(4, 900, torch.float32)
    check(x, x.argmax(-1), 3)


def test_shapes_and_views():
    x = _logits(12, 1001, torch.bfloat16)
    tokens = _tokens(12, 1001)
    want = check(x, tokens, 2)
    got = score.token_scores(x.view(3, 4, 1001), tokens.view(3, 4), top=2)
    assert got.logprob.shape == (3, 4) and got.top_token.shape == (3, 4, 2)
    assert all(torch.equal(a.flatten(0, 1), b) for a, b in zip(got, want))
    one = score.token_scores(x[5], tokens[5], top=2)
    assert one.logprob.shape == () and one.top_token.shape == (2,) and torch.equal(one.top_token, want.top_token[5])
    wide = torch.empty(12, 1203, dtype=torch.bfloat16, device="cuda")
    wide[:, 101:1102] = x
    views = [wide[:, 101:1102], x.t().contiguous().t(), x[:1].expand(12, 1001)]
    for v in views[:2]:
        assert all(torch.equal(a, b) for a, b in zip(score.token_scores(v, tokens, top=2), want))
    for v in views:
        leaf = v.detach().requires_grad_()
        r = score.token_scores(leaf, tokens, top=2)
        (dx,) = torch.autograd.grad(r.logprob.sum(), leaf)
        ref = scores(v, tokens, 2, torch.ones(12).cuda(), torch.zeros(12).cuda(), torch.zeros(12, 2).cuda())
        tol = score_tolerances(v, ref, torch.ones(12).cuda(), torch.zeros(12).cuda(), torch.zeros(12, 2).cuda())
        within(dx, ref[4], tol[3], "gradient")
    apart = torch.stack((tokens, tokens), 1)[:, 0]
    assert torch.equal(score.token_scores(x, apart).logprob, want.logprob)
    none = score.token_scores(x[:0], tokens[:0], top=2)
    assert none.logprob.shape == (0,) and none.top_token.shape == (0, 2)
    leaf = x[:0].clone().requires_grad_()
    (dx,) = torch.autograd.grad(score.token_scores(leaf, tokens[:0]).logprob.sum(), leaf)
    assert dx.shape == (0, 1001)


def test_gradients_against_differences():
    x = _logits(2, 11, torch.float32, spread=1.0)
    tokens = torch.tensor([4, 0]).cuda()

    def f(x):
        r = score.token_scores(x, tokens, top=2)
        return (r.logprob * 0.7 - r.entropy * 1.3).double().sum() + (r.top_logprob.double() * torch.tensor([0.5, -2.0]).cuda()).sum()

    leaf = x.clone().requires_grad_()
    (dx,) = torch.autograd.grad(f(leaf), leaf)
    h = 2.0**-9
    for i in range(22):
        ends = []
        for step in (h, -h):
            y = x.clone()
            y.view(-1)[i] += step
            ends.append(float(f(y)))
        assert abs((ends[0] - ends[1]) / (2 * h) - float(dx.view(-1)[i])) < 2e-3


def test_in_a_graph_and_on_another_stream():
    x = _logits(3, 70000, torch.bfloat16).requires_grad_()
    tokens = _tokens(3, 70000)

    def step():
        r = score.token_scores(x, tokens, top=3)
        (dx,) = torch.autograd.grad(r.logprob.sum() - r.entropy.sum(), x)
        return [y.detach() for y in r] + [dx]

    want = step()
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        got = step()
    torch.cuda.current_stream().wait_stream(s)
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step()
    other = _tokens(3, 70000, seed=5)
    for k in range(3):
        tokens.copy_(other if k == 1 else _tokens(3, 70000))
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, step()))


FAR = [(d, f) for d in DTYPES for f in (-40000.0, 300.0, 65500.0, 65537.0, 1e6) if f <= torch.finfo(d).max]


@pytest.mark.parametrize("dtype,far", FAR)
def test_far_maxima(dtype, far):
    """Rows about a far value: exponents are differences, on both sides of 2^16,
    from which on they are found in another way."""
    for vocab in (1000, 50257):
        x = (_logits(3, vocab, torch.float32) + far).clamp(max=torch.finfo(dtype).max).to(dtype)
        check(x, _tokens(3, vocab), 0)
        check(x, _tokens(3, vocab), 5)
