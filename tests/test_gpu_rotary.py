"""Rotary positions on the GPU against complex numbers in float64."""

import math

import pytest
import torch

from draft_helpers import turn_tolerance, turned
from voyager_amd import rotary

pytestmark = pytest.mark.gpu
DTYPES = [torch.bfloat16, torch.float16, torch.float32]


def _check(rot, got, x, positions, back=False):
    f, factor = rotary.frequencies(rot.rotary_dim, rot.theta_, rot.scaling_)
    how = (rot.rotary_dim, rot.interleaved)
    ref = turned(x.detach().cpu(), positions.cpu(), f, factor, *how, back=back)
    tol = turn_tolerance(x.detach().cpu(), ref, factor, *how)
    bad = (got.detach().cpu().double() - ref).abs() > tol
    assert got.is_contiguous() and got.dtype == x.dtype
    assert not bool(bad.any()), f"{int(bad.sum())} of {bad.numel()} beyond the tolerance"


def _rot(dim, theta=1e4, scaling=None, **kw):
    r = rotary.Rotary(dim, theta=theta, scaling=scaling, **kw)
    r.theta_, r.scaling_ = theta, scaling
    return r


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("b,t,heads,kv,dim,rotary_dim", [
    (1, 1, 32, 8, 128, 128), (2, 5, 3, 1, 64, 32), (1, 1030, 2, 2, 64, 64), (3, 7, 1, 1, 80, 20), (1, 3, 5, 5, 6, 2),
    (2, 2, 2, 1, 512, 512), (1, 2, 300, 1, 96, 96), (1, 1025, 1, 1, 10, 10)])
def test_values(dtype, interleaved, b, t, heads, kv, dim, rotary_dim):
    g = torch.Generator().manual_seed(dim + t)
    rot = _rot(dim, rotary_dim=rotary_dim, interleaved=interleaved)
    q = torch.randn(b, t, heads, dim, generator=g).to(dtype).cuda()
    k = torch.randn(b, t, kv, dim, generator=g).to(dtype).cuda()
    pos = torch.randint(0, 5000, (b, t), generator=g).cuda()
    for p in (pos, pos.int()):
        qo, ko = rot(q, k, p)
        _check(rot, qo, q, pos)
        _check(rot, ko, k, pos)
    assert torch.equal(qo[..., rotary_dim:], q[..., rotary_dim:])


@pytest.mark.parametrize("scaling", [None, {"kind": "linear", "factor": 4.0}, {"kind": "ntk", "factor": 4.0},
                                     {"kind": "bands", "factor": 8.0, "low": 1.0, "high": 4.0, "trained": 8192},
                                     {"kind": "yarn", "factor": 16.0, "low": 1.0, "high": 32.0, "trained": 4096}])
def test_far_positions(scaling):
    """Positions past 2^24, and negative ones: the angle is not a float32's."""
    rot = _rot(128, theta=5e5, scaling=scaling)
    q = torch.randn(1, 6, 2, 128, generator=torch.Generator().manual_seed(1)).cuda()
    pos = torch.tensor([0, 1, 999_999, 2**24 + 1, 2**31 - 1, -12345]).cuda()
    qo, ko = rot(q, None, pos)
    assert ko is None
    _check(rot, qo, q, pos[None])


def test_views_and_shared_positions():
    g = torch.Generator().manual_seed(2)
    rot = _rot(64)
    fused = torch.randn(2, 9, 8, 64, generator=g).bfloat16().cuda()
    q, k = fused[:, :, :4], fused[:, :, 4:6]
    pos = torch.arange(100, 109).cuda()
    shapes = [(q, k), (q.transpose(1, 2).contiguous().transpose(1, 2), k)]  # tokens last but one; heads first in memory
    odd = torch.empty(2, 9, 4, 67, dtype=torch.bfloat16, device="cuda")[..., 1:65]  # rows 2 bytes off 16
    odd.copy_(q)
    shapes.append((odd, k))
    shapes.append((q.contiguous().transpose(2, 3).contiguous().transpose(2, 3), k))  # channels not dense
    first = None
    for qq, kk in shapes:
        for p in (pos, pos[None], pos[None].expand(2, 9), torch.stack((pos, pos)).t().contiguous().t()):
            qo, ko = rot(qq, kk, p)
            if first is None:
                first = (qo, ko)
                _check(rot, qo, q, pos[None].expand(2, 9))
            assert torch.equal(qo, first[0]) and torch.equal(ko, first[1])
    none, ko = rot(None, k, pos)
    assert none is None and torch.equal(ko, first[1])


def test_nothing_and_nan():
    rot = _rot(8)
    for b, t, h in ((0, 3, 2), (2, 0, 2), (2, 3, 0)):
        q = torch.zeros(b, t, h, 8, device="cuda")
        assert rot(q, None, torch.arange(t).cuda())[0].shape == q.shape
    q = torch.tensor([math.nan, math.inf, 1.0, 2.0, 3.0, 4.0, 5.0, 6.0], device="cuda").reshape(1, 1, 1, 8)
    qo, _ = rot(q, None, torch.tensor([3]).cuda())
    bad = ~torch.isfinite(qo.flatten().cpu())
    assert bad.tolist() == [True, True, False, False, True, True, False, False]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("interleaved", [False, True])
def test_gradient_is_the_turn_back(dtype, interleaved):
    g = torch.Generator().manual_seed(3)
    rot = _rot(32, rotary_dim=16, interleaved=interleaved, scaling={"kind": "yarn", "factor": 4.0, "low": 1.0,
                                                                      "high": 8.0, "trained": 64})
    q = torch.randn(2, 5, 3, 32, generator=g).to(dtype).cuda().requires_grad_()
    k = torch.randn(2, 5, 1, 32, generator=g).to(dtype).cuda().requires_grad_()
    pos = torch.randint(0, 300, (2, 5), generator=g).cuda()
    gq = torch.randn(2, 5, 3, 32, generator=g).to(dtype).cuda()
    gk = torch.randn(2, 5, 1, 32, generator=g).to(dtype).cuda()
    dq, dk = torch.autograd.grad(rot(q, k, pos), (q, k), (gq, gk))
    _check(rot, dq, gq, pos, back=True)
    _check(rot, dk, gk, pos, back=True)
    # one of them alone, and an output that nothing follows
    (only,) = torch.autograd.grad(rot(q, k, pos)[0], (q,), (gq,))
    assert torch.equal(only, dq)
    (only,) = torch.autograd.grad(rot(q.detach(), k, pos)[1], (k,), (gk,))
    assert torch.equal(only, dk)


def test_gradient_against_differences():
    """The operator is linear: (f(x + h d) - f(x - h d)) / 2h is its value at d
    up to float32's rounding, for any h."""
    g = torch.Generator().manual_seed(4)
    rot = _rot(16, interleaved=True)
    x, d, w = (torch.randn(1, 4, 2, 16, generator=g).cuda() for _ in range(3))
    pos = torch.arange(4).cuda()
    x.requires_grad_()
    (grad,) = torch.autograd.grad((rot(x, None, pos)[0] * w).sum(), x)
    f = lambda y: (rot(y, None, pos)[0].double() * w.double()).sum()
    with torch.no_grad():
        slope = (f(x + 0.5 * d) - f(x - 0.5 * d)) / 1.0
    want = (grad.double() * d.double()).sum()
    # each of 128 outputs within 12 half steps of values up to about 5, times weights up to about 4
    assert abs(float(slope - want)) <= 128 * 12 * 2.0**-24 * 5 * 4
    # and of the gradient: the same turn again
    y = torch.randn(1, 4, 2, 16, generator=g).cuda().requires_grad_()
    (gx,) = torch.autograd.grad(rot(x, None, pos)[0], x, y, create_graph=True)
    (gy,) = torch.autograd.grad(gx, y, w)
    assert torch.equal(gy, rot(w, None, pos)[0])


def test_captured_with_its_gradient():
    rot = _rot(64)
    g = torch.Generator().manual_seed(5)
    q = torch.randn(1, 8, 4, 64, generator=g).bfloat16().cuda()
    k = torch.randn(1, 8, 2, 64, generator=g).bfloat16().cuda()
    pos = torch.arange(8).cuda()

    def step():
        a, b = q.detach().requires_grad_(), k.detach().requires_grad_()  # leaves of this graph alone
        out = rot(a, b, pos)
        return [*(o.detach() for o in out), *torch.autograd.grad(out, (a, b), (q, k))]

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step()
    for i in range(3):
        q.copy_(torch.randn(q.shape, generator=g))
        pos.add_(1000 * i)
        exp = step()
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, exp)), f"replay {i}"
