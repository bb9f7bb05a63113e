"""Norms of queries and keys with rotary positions on the GPU, and their
gradients, against float64."""

import pytest
import torch

from pass_helpers import norm_turned, norm_turned_back, within
from voyager_amd import rotary

pytestmark = pytest.mark.gpu
DTYPES = [torch.bfloat16, torch.float16, torch.float32]
SCALING = {"kind": "yarn", "factor": 16.0, "low": 1.0, "high": 32.0, "trained": 4096}


class Case:
    def __init__(self, b, t, heads, kv, dim, rotary_dim=None, dtype=torch.bfloat16, weights=None, interleaved=False,
                 scaling=None, eps=1e-6, seed=0):
        g = torch.Generator().manual_seed(seed + dim + t)
        self.rot = rotary.Rotary(dim, theta=1e4, rotary_dim=rotary_dim, interleaved=interleaved, scaling=scaling)
        f, factor = rotary.frequencies(self.rot.rotary_dim, 1e4, scaling)
        self.how, self.eps = (f, factor, self.rot.rotary_dim, interleaved), eps
        n = lambda *s: torch.randn(*s, generator=g)
        self.q, self.k = ((n(b, t, h, dim) * torch.exp(n(b, t, h, 1))).to(dtype).cuda() for h in (heads, kv))
        self.gq, self.gk = (n(b, t, h, dim).to(dtype).cuda() for h in (heads, kv))
        self.qw, self.kw = ((1 + 0.3 * n(dim)).to(weights or dtype).cuda() for _ in range(2))
        self.pos = torch.randint(0, 100000, (b, t), generator=g).cuda()

    def run(self, q, k, pos=None, qw=None, kw=None):
        return self.rot.normed(q, k, self.pos if pos is None else pos, self.qw if qw is None else qw,
                               self.kw if kw is None else kw, eps=self.eps)

    def check_values(self, got):
        for y, x, w in ((got[0], self.q, self.qw), (got[1], self.k, self.kw)):
            assert y.is_contiguous() and y.dtype == x.dtype
            within(y, *norm_turned(x.cpu(), w.cpu(), self.pos.cpu(), *self.how, self.eps), "values")

    def check_grads(self, grads):
        for (dx, dw), x, w, g in ((grads[:2], self.q, self.qw, self.gq), (grads[2:], self.k, self.kw, self.gk)):
            rx, rw, tx, tw = norm_turned_back(x.cpu(), w.cpu(), g.cpu(), self.pos.cpu(), *self.how, self.eps)
            assert dx.dtype == x.dtype and dw.dtype == w.dtype
            within(dx, rx, tx, "inputs' gradient")
            within(dw, rw, tw, "weights' gradient")

    def leaves(self):
        return [t.clone().requires_grad_() for t in (self.q, self.qw, self.k, self.kw)]

    def grads(self):
        q, qw, k, kw = leaves = self.leaves()
        return torch.autograd.grad(self.run(q, k, qw=qw, kw=kw), leaves, (self.gq, self.gk))


SHAPES = [(1, 1, 32, 8, 128, 128), (2, 5, 3, 1, 64, 32), (1, 2050, 2, 1, 64, 64), (3, 7, 1, 1, 80, 20), (1, 3, 5, 5, 6, 2),
          (2, 2, 2, 1, 512, 512), (1, 2, 300, 1, 96, 96), (1, 1025, 1, 1, 10, 10), (1, 3, 2, 2, 2, 2), (1, 4, 8, 2, 256, 256),
          (1, 3, 2, 1, 510, 254)]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("shape", SHAPES)
def test_values_and_gradients(dtype, interleaved, shape):
    c = Case(*shape[:5], rotary_dim=shape[5], dtype=dtype, interleaved=interleaved)
    c.check_values(c.run(c.q, c.k))
    c.check_grads(c.grads())


@pytest.mark.parametrize("dtype", DTYPES[:2])
def test_float32_weights_and_a_factor(dtype):
    c = Case(1, 37, 4, 2, 128, dtype=dtype, weights=torch.float32, scaling=SCALING)
    c.check_values(c.run(c.q, c.k))
    c.check_grads(c.grads())


def test_many_tokens_share_the_weights_gradient():
    """More tokens than workgroups take at a time: sums of many rounds, the same each time."""
    c = Case(2, 3001, 3, 2, 64)
    a, b = c.grads(), c.grads()
    c.check_grads(a)
    assert all(torch.equal(x, y) for x, y in zip(a, b))


def test_more_rows_and_heads_than_workgroups():
    """The last rows, and the last heads, beside a call of their own."""
    for b, t, heads, dim in ((1, (1 << 26) + 5, 1, 2), (1, 2, 300000, 130)):
        rot = rotary.Rotary(dim)
        g = torch.Generator(device="cuda").manual_seed(t + heads)
        q = torch.randn(b, t, heads, dim, generator=g, device="cuda", dtype=torch.bfloat16)
        w = torch.linspace(0.5, 1.5, dim, device="cuda")
        pos = torch.arange(t, device="cuda", dtype=torch.int32)
        rows, of = min(t, 1000), min(heads, 100)
        y = rot.normed(q, None, pos, w, None)[0]
        assert torch.equal(y[:, -rows:, -of:], rot.normed(q[:, -rows:, -of:], None, pos[-rows:], w, None)[0])
        assert torch.equal(y[:, :rows, :of], rot.normed(q[:, :rows, :of], None, pos[:rows], w, None)[0])
        x = q.requires_grad_()
        go = torch.ones((), device="cuda", dtype=torch.bfloat16).expand(q.shape)
        dx, = torch.autograd.grad(rot.normed(x, None, pos, w, None)[0], x, go)
        part = q.detach()[:, -rows:, -of:].requires_grad_()
        dp, = torch.autograd.grad(rot.normed(part, None, pos[-rows:], w, None)[0], part, go[:, -rows:, -of:])
        assert torch.equal(dx[:, -rows:, -of:], dp)


def test_views():
    c = Case(2, 9, 4, 2, 64)
    fused = torch.cat((c.q, c.k, c.k), 2)
    y = c.run(fused[:, :, :4], fused[:, :, 4:6])
    c.check_values(y)
    odd = torch.empty(2, 9, 4, 67, dtype=torch.bfloat16, device="cuda")[..., 1:65]  # rows 2 bytes off 16
    odd.copy_(c.q)
    turned_round = c.q.transpose(2, 3).contiguous().transpose(2, 3)  # channels not dense
    weight = torch.stack((c.qw, c.qw), 1)[:, 0]
    for q in (odd, turned_round):
        got = c.run(q, c.k, qw=weight)
        c.check_values(got)
    for g in (torch.cat((c.gq, c.gq), 3)[..., :64], c.gq.transpose(1, 2).contiguous().transpose(1, 2), odd.copy_(c.gq)):
        leaves = c.leaves()
        q, qw, k, kw = leaves
        c.check_grads(torch.autograd.grad(c.run(q, k, qw=qw, kw=kw), leaves, (g, c.gk)))


def test_a_gradient_of_one_value_for_all():
    c = Case(1, 5, 2, 2, 64)
    c.gq, c.gk = torch.ones_like(c.gq), torch.ones_like(c.gk)
    leaves = c.leaves()
    q, qw, k, kw = leaves
    a, b = c.run(q, k, qw=qw, kw=kw)
    c.check_grads(torch.autograd.grad(a.sum() + b.sum(), leaves))


def test_one_tensor_and_partial_gradients():
    c = Case(1, 6, 4, 2, 64)
    whole = c.grads()
    y, none = c.rot.normed(c.q, None, c.pos, c.qw, None, eps=c.eps)
    assert none is None
    none, z = c.rot.normed(None, c.k, c.pos, None, c.kw, eps=c.eps)
    assert none is None
    c.check_values((y, z))
    q, qw, k, kw = c.leaves()
    a, b = c.run(q, k, qw=qw, kw=kw)
    got = torch.autograd.grad(a, (q, qw, k, kw), c.gq, allow_unused=True, retain_graph=True)
    assert torch.equal(got[0], whole[0]) and torch.equal(got[1], whole[1]) and got[2] is None and got[3] is None
    got = torch.autograd.grad(b, (k, kw), c.gk)
    assert torch.equal(got[0], whole[2]) and torch.equal(got[1], whole[3])
    a, b = c.run(c.q, k, kw=kw)  # weights and inputs that need none
    got = torch.autograd.grad((a, b), (k, kw), (c.gq, c.gk)) if a.requires_grad else None
    assert torch.equal(got[0], whole[2]) and torch.equal(got[1], whole[3])
    a, b = c.run(q, k)
    assert torch.equal(torch.autograd.grad((a, b), (q, k), (c.gq, c.gk))[0], whole[0])
    a, b = c.run(c.q, c.k, qw=qw, kw=kw)
    assert torch.equal(torch.autograd.grad((a, b), (qw, kw), (c.gq, c.gk))[1], whole[3])


def test_no_second_gradient():
    c = Case(1, 2, 2, 1, 64)
    leaves = c.leaves()
    q, qw, k, kw = leaves
    with pytest.raises(RuntimeError, match="differentiable once"):
        torch.autograd.grad(c.run(q, k, qw=qw, kw=kw), leaves, (c.gq, c.gk), create_graph=True)


def test_gradients_against_differences():
    c = Case(1, 2, 2, 1, 8, rotary_dim=4, dtype=torch.float32)
    leaves = c.leaves()

    def f(q, qw, k, kw):
        a, b = c.run(q, k, qw=qw, kw=kw)
        return (a.double() * c.gq).sum() + (b.double() * c.gk).sum()

    grads = torch.autograd.grad(f(*leaves), leaves)
    h = 2.0**-7
    for i, leaf in enumerate(leaves):
        for at in range(0, leaf.numel(), 5):
            ends = []
            for step in (h, -h):
                moved = [x.detach().clone() for x in leaves]
                moved[i].view(-1)[at] += step
                ends.append(float(f(*moved)))
            # a difference's error: the third derivative's h^2, and float32's of the values over h
            assert abs((ends[0] - ends[1]) / (2 * h) - float(grads[i].view(-1)[at])) < 2e-2 * (1 + float(grads[i].abs().max()))


def test_rows_of_nothing_and_nothing_at_all():
    c = Case(1, 4, 2, 1, 64, dtype=torch.float32)
    c.q[:, 1] = 0
    c.q[:, 2] = torch.tensor(2.0**-80)
    c.check_values(c.run(c.q, c.k))
    c.check_grads(c.grads())
    e = Case(1, 0, 2, 1, 64)
    y, z = e.run(e.q, e.k)
    assert y.shape == (1, 0, 2, 64) and z.shape == (1, 0, 1, 64)
    grads = e.grads()
    assert not grads[1].any() and not grads[3].any() and grads[0].shape == e.q.shape


def test_a_bad_row_stays_its_own():
    c = Case(1, 4, 2, 1, 64)
    good = c.run(c.q, c.k)[0]
    bad = c.q.clone()
    bad[0, 1, 0, 3], bad[0, 2, 1, 5] = float("nan"), float("inf")
    y = c.run(bad, c.k)[0]
    same = torch.ones(1, 4, 2, dtype=torch.bool)
    same[0, 1, 0] = same[0, 2, 1] = False
    assert torch.equal(y[same], good[same]) and bool(torch.isnan(y[0, 1, 0]).all()) and not bool(torch.isfinite(y[0, 2, 1, 5]))


def test_in_a_graph_and_on_another_stream():
    c = Case(2, 33, 4, 2, 128)
    want = [*c.run(c.q, c.k), *c.grads()]
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    leaves = c.leaves()
    q, qw, k, kw = leaves

    def step():
        y = c.run(q, k, qw=qw, kw=kw)
        return [x.detach() for x in y] + list(torch.autograd.grad(y, leaves, (c.gq, c.gk)))

    with torch.cuda.stream(s):
        got = step()
    torch.cuda.current_stream().wait_stream(s)
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step()
    for _ in range(3):
        for x in got:
            x.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, want))
        assert all(torch.equal(a, b) for a, b in zip(step(), want))
