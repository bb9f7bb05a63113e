"""Causal attention of packed sequences on the GPU, and its gradients, against float64."""

import math

import pytest
import torch

from pass_helpers import packed_attention, within
from voyager_amd import prompt

pytestmark = pytest.mark.gpu
BF16, F16 = torch.bfloat16, torch.float16


def offsets_of(lengths):
    at = [0]
    for n in lengths:
        at.append(at[-1] + n)
    return at


class Case:
    def __init__(self, lengths, heads, kv, d, dtype, pad=0, scale=None, seed=0, spread=0.5):
        self.offsets = offsets_of(lengths)
        n = self.offsets[-1] + pad
        g = torch.Generator().manual_seed(seed + n + heads + d)
        r = lambda h: (torch.randn(n, h, d, generator=g) * torch.exp(spread * torch.randn(1, h, 1, generator=g))).to(dtype).cuda()
        self.q, self.k, self.v, self.go = r(heads), r(kv), r(kv), r(heads)
        self.scale = d ** -0.5 if scale is None else scale
        self.packing = prompt.Packing(torch.tensor(self.offsets, dtype=torch.int32).cuda(), n)

    def run(self, q=None, k=None, v=None, go=None):
        leaves = [t.detach().requires_grad_() for t in (self.q if q is None else q, self.k if k is None else k, self.v if v is None else v)]
        o, lse = prompt.prompt_attention(*leaves, self.packing, scale=self.scale, return_lse=True)
        return [o.detach(), lse, *torch.autograd.grad(o, leaves, self.go if go is None else go)]

    def check(self, got=None, which=slice(0, 5)):
        got = self.run() if got is None else got
        ref, tol = packed_attention(self.q, self.k, self.v, self.offsets, self.scale, self.go)
        for y, r, e, name in list(zip(got, ref, tol, ("output", "lse", "dq", "dk", "dv")))[which]:
            if name == "lse":
                empty = torch.isinf(r)
                assert torch.equal(y == -math.inf, empty)
                y, r = y.masked_fill(empty, 0), r.masked_fill(empty, 0)
            else:
                assert y.is_contiguous() and y.dtype == self.q.dtype
                # a value past the type's largest, 65504 in float16, is rounded to an infinity of its sign
                past = (r.abs() + e >= torch.finfo(y.dtype).max) & (y == torch.sign(r) * math.inf)
                y, r = y.double().masked_fill(past, 0), r.masked_fill(past, 0)
            within(y, r, e, name)
        return got


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("lengths,pad,heads,kv", [
    ([1], 0, 1, 1), ([2], 0, 2, 1), ([33], 0, 4, 2), ([128], 0, 2, 2), ([129], 5, 3, 1), ([31, 1, 0, 96], 0, 2, 2),
    ([0, 0, 65, 64, 63, 0], 40, 2, 1), ([300], 0, 7, 1), ([1] * 150, 0, 2, 1), ([100, 200, 5, 1, 260], 130, 8, 4),
    ([700], 3, 2, 2)])
def test_values_and_gradients(dtype, d, lengths, pad, heads, kv):
    Case(lengths, heads, kv, d, dtype, pad).check()


@pytest.mark.parametrize("dtype,d", [(BF16, 128), (F16, 64), (BF16, 256)])
def test_long_sequences_are_cut_for_the_keys(dtype, d):
    """Blocks of keys that many rows see are cut into items whose sums are joined; a short sequence beside a long one is not."""
    Case([2900, 40, 3, 500], 2, 1, d, dtype, 77).check()


@pytest.mark.parametrize("dtype,d", [(F16, 128), (BF16, 64), (BF16, 256)])
def test_a_long_sequence_among_many_short_ones(dtype, d):
    """By the mean they are short; the long one's blocks are cut all the same."""
    Case([3] * 20 + [1700, 0, 9], 2, 1, d, dtype, 40).check()


@pytest.mark.parametrize("dtype", [BF16, F16])
def test_more_blocks_than_are_cut(dtype):
    c = Case([60] * 1500 + [700], 24, 12, 64, dtype, 9)
    assert (c.packing.tokens + 127) // 128 * 12 > 4096
    got = c.run()
    a, b = c.offsets[-4], c.offsets[-1]  # the last three sequences, as a batch of their own
    ref, tol = packed_attention(*(t[a:b] for t in (c.q, c.k, c.v)), [0, 60, 120, 820], c.scale, c.go[a:b])
    for y, r, e in zip(got, ref, tol):
        within(y[a:b], r, e)


@pytest.mark.parametrize("dtype,d", [(BF16, 128), (F16, 64), (F16, 256)])
def test_sharp_and_scaled_scores(dtype, d):
    Case([200, 77], 2, 1, d, dtype, scale=1.0, spread=0.3).check()  # a key or two take all
    Case([200, 77], 2, 1, d, dtype, scale=1e-3).check()
    c = Case([150], 2, 1, d, dtype)
    c.k[:75] *= 8  # the largest scores come first, then only small ones
    c.check()
    c.k = c.k.flip(0).contiguous()  # and the other way round: the reference rises
    c.check()


@pytest.mark.parametrize("d", [64, 128, 256])
def test_views(d):
    c = Case([90, 60], 4, 2, d, BF16, 7)
    want = c.check()
    n = c.packing.tokens
    fused = torch.cat((c.q, c.k, c.v), 1)
    parts = fused[:, :4], fused[:, 4:6], fused[:, 6:]
    heads_first = [t.transpose(0, 1).contiguous().transpose(0, 1) for t in (c.q, c.k, c.v)]
    odd = []
    for t in (c.q, c.k, c.v):  # rows 2 bytes off 16, which are copied
        x = torch.empty(n, t.shape[1], d + 3, dtype=BF16, device="cuda")[..., 1:d + 1]
        odd.append(x.copy_(t))
    turned = [t.transpose(1, 2).contiguous().transpose(1, 2) for t in (c.q, c.k, c.v)]
    off = [torch.cat((t.flatten()[:3], t.flatten()))[3:].view(t.shape) for t in (c.q, c.k, c.v)]  # dense, but off 16 bytes
    for q, k, v in (parts, heads_first, odd, turned, off):
        assert all(torch.equal(a, b) for a, b in zip(c.run(q, k, v), want))
    for go in (torch.cat((c.go, c.go), 1)[:, :4], c.go.transpose(0, 1).contiguous().transpose(0, 1),
               c.go.transpose(1, 2).contiguous().transpose(1, 2)):
        assert all(torch.equal(a, b) for a, b in zip(c.run(go=go), want))
    one = c.k[:, :1].expand(n, 2, d)  # a head's keys for both
    got = c.run(k=one)
    c.k = one.contiguous()
    c.check(got)


@pytest.mark.parametrize("dtype,d", [(BF16, 64), (F16, 128), (BF16, 256)])
@pytest.mark.parametrize("lengths", [[40], [300, 7], [700]])
def test_far_scores_of_one_key(dtype, d, lengths):
    """Each row is its own key's alone, with a score of some thousands, whose
    logarithm of a sum float32 holds to 2^-11 only: the scores' gradients are 0.
    A weight's gradient and D are two sums of at most 256 products, each off by at
    most 2^-16 of the sum of their magnitudes, and what o and its remainder leave
    out by 2^-18: together under 2^-14."""
    c = Case(lengths, 2, 2, d, dtype, scale=1.0)
    c.k = (8192 ** 0.5 * torch.nn.functional.normalize(c.k.float(), dim=2)).to(dtype)
    _, lse, dq, dk, _ = c.run(q=c.k)
    assert 8000 < float(lse.min()) and float(lse.max()) < 8400
    most = 2.0 ** -14 * (c.go.double() * c.v.double()).abs().sum(2, keepdim=True) * c.k.double().abs()
    for name, y in (("dq", dq), ("dk", dk)):
        assert bool((y.double().abs() <= most).all()), (name, float((y.double().abs() / most).max()))


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("lengths", [[2], [1, 3, 1], [40], [300, 17]])
def test_gradients_of_short_sequences_are_rounded_once(dtype, d, lengths):
    """A result's rounding is off by half a step at most, by a fifth of that and
    more on average: 2^-11 of it in bfloat16, 2^-14 in float16.  Weights and their
    gradients in two parts are off by 2^-18 and 2^-22, float32 sums of at most 300
    products by some 2^-20 of their magnitudes: under a quarter of it in both, added in squares 1.04."""
    c = Case(lengths, 3, 1, d, dtype)
    ref, _ = packed_attention(c.q, c.k, c.v, c.offsets, c.scale, c.go)
    for y, r, name in list(zip(c.run(), ref, ("output", "lse", "dq", "dk", "dv")))[2:]:
        once = (r.to(dtype).double() - r).norm()
        assert float((y.double() - r).norm()) <= float(once) * 1.04 + 1e-9, name


def test_a_gradient_of_one_value_for_all():
    c = Case([70, 30], 2, 1, 64, F16)
    c.go = torch.ones_like(c.go)
    leaves = [t.detach().requires_grad_() for t in (c.q, c.k, c.v)]
    o = prompt.prompt_attention(*leaves, c.packing)
    want = c.check()
    assert all(torch.equal(a, b) for a, b in zip(torch.autograd.grad(o.sum(), leaves), want[2:]))


@pytest.mark.parametrize("dtype,d", [(BF16, 128), (F16, 128), (BF16, 64), (F16, 256)])
@pytest.mark.parametrize("bad", [math.nan, math.inf, -math.inf])
@pytest.mark.parametrize("lengths", [(70, 41, 90), (600, 41, 900)])  # the second: by two halves of a workgroup
def test_what_is_not_seen_has_no_part(dtype, d, bad, lengths):
    """Infinities and NaN in a sequence's last row, in the rows that pad and
    in q, k, v and the result's gradient there: earlier rows and other sequences are as
    they were, bit for bit, and so are the keys that these rows do not see."""
    c = Case(lengths, 4, 2, d, dtype, 20)
    want = c.check()
    n, third = c.offsets[-1], c.offsets[2]
    for what in ("q", "k", "v", "go"):
        for rows in ([third - 1], [n - 1], list(range(n, n + 20)), [30, third + 39]):
            t = {x: getattr(c, x).clone() for x in ("q", "k", "v", "go")}
            for r in rows:
                t[what][r, 1, 5] = bad
                t[what][r, 0] = bad
            got = c.run(**t)
            touched = torch.zeros(n + 20, dtype=torch.bool)  # rows and keys that may show it
            seen = torch.zeros(n + 20, dtype=torch.bool)
            for r in rows:
                for a, b in zip(c.offsets, c.offsets[1:]):
                    if a <= r < b:
                        if what in ("q", "go"):
                            touched[r] = True
                            seen[a:r + 1] = True
                        else:  # keys: the rows from there on, and the keys that those rows see
                            touched[r:b] = True
                            seen[a:b] = True
            for i, y in enumerate(got):
                bad_rows = (touched if i < 3 else seen)
                if what == "go" and i < 2:
                    bad_rows = torch.zeros_like(touched)
                same = ~bad_rows.cuda()
                assert torch.equal(y[same], want[i][same]), (what, rows, i)
            inside = [r for r in rows if r < n]
            if inside and what != "go":
                assert not bool(torch.isfinite(got[0][inside]).all())


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("pad", [0, 600])  # rows enough for two halves of a workgroup
def test_an_infinite_value_gives_its_channel_an_infinity(dtype, d, pad):
    c = Case([150], 2, 1, d, dtype, pad)
    clean = c.run()[0]
    v = c.v.clone()
    v[100, 0, 7], v[140, 0, 9] = math.inf, -math.inf
    o = c.run(v=v)[0]
    assert bool((o[100:150, :, 7] == math.inf).all()) and bool((o[140:150, :, 9] == -math.inf).all())
    o[100:150, :, 7], o[140:150, :, 9] = clean[100:150, :, 7], clean[140:150, :, 9]
    assert torch.equal(o, clean)
    v[120, 0, 7] = -math.inf
    o = c.run(v=v)[0]
    assert bool((o[100:120, :, 7] == math.inf).all()) and bool(torch.isnan(o[120:150, :, 7]).all())


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("lengths", [(300, 40), (1000, 40)])
def test_the_largest_values_give_finite_results(dtype, lengths):
    c = Case(lengths, 2, 1, 128, dtype)
    most = torch.finfo(dtype).max
    c.v = torch.where(c.v > 0, most, -most).to(dtype)
    c.check(which=slice(0, 2))
    c.v = torch.full_like(c.v, most)
    o = c.run()[0]
    assert bool((o == most).all())


@pytest.mark.parametrize("length", [500, 1100])  # the second: by two halves of a workgroup
@pytest.mark.parametrize("size", [2.0**-14, 2.0**10])
def test_small_and_large_gradients_in_float16(size, length):
    """Gradients of weights that float16 could not hold as they come: under its
    least value, or, where values are large as well, over its largest."""
    c = Case([length, 30], 2, 1, 64, F16)
    c.go = (c.go * 0 + 1) * torch.randn(c.go.shape, generator=torch.Generator().manual_seed(1)).cuda() * size
    c.go = c.go.to(F16)
    if size > 1:
        c.v = (c.v * 64).to(F16)
        c.k, c.q = (c.k / 64).to(F16), (c.q / 64).to(F16)
        c.scale = 64.0
    c.check()
    one = Case([4, 200], 2, 1, 64, F16)
    one.go[:4] *= 2.0**-13  # a sequence's are small beside the next one's
    one.check()


def test_gradients_against_differences():
    """Along the gradient itself, the difference of the kernel's own sums.  A result is off by its
    rounding, at most 2^-11 of itself, and by as much from the rounded weights."""
    c = Case([5, 9], 2, 1, 64, F16, spread=0.1)
    grads = c.run()[2:]
    inputs = {"q": c.q, "k": c.k, "v": c.v}
    for (name, x), g in zip(inputs.items(), grads):
        u = g.double() / g.double().norm()
        ends, moved = [], []
        for sign in (1, -1):
            y = (x.double() + sign * 0.25 * u).to(F16)
            moved.append(y.double())
            with torch.no_grad():
                o = prompt.prompt_attention(**{**inputs, name: y}, packing=c.packing)
            ends.append((o.double() * c.go.double()).sum())
            noise = (o.double().abs() * c.go.double().abs()).sum() * 2.0**-11 * 2
        want = ((moved[0] - moved[1]) * g.double()).sum()
        # and the third derivative's, a 64th of the step's square at these sizes
        assert abs(float(ends[0] - ends[1] - want)) < float(2 * noise + 0.02 * want.abs())


def test_the_same_every_time():
    c = Case([1700, 300, 90], 8, 2, 128, BF16, 11)
    first = c.run()
    for _ in range(3):
        assert all(torch.equal(a, b) for a, b in zip(c.run(), first))


def test_without_gradients_and_some_gradients():
    c = Case([40, 50], 2, 1, 64, BF16)
    want = c.run()
    with torch.no_grad():
        o = prompt.prompt_attention(c.q, c.k, c.v, c.packing)
    assert torch.equal(o, want[0]) and not o.requires_grad
    q = c.q.clone().requires_grad_()
    (gq,) = torch.autograd.grad(prompt.prompt_attention(q, c.k, c.v, c.packing), q, c.go)
    assert torch.equal(gq, want[2])
    o, lse = prompt.prompt_attention(q, c.k, c.v, c.packing, return_lse=True)
    assert not lse.requires_grad
    with pytest.raises(RuntimeError, match="differentiable once"):
        torch.autograd.grad(o, q, c.go, create_graph=True)


def test_bad_offsets_pad_everything():
    q, k = torch.randn(50, 2, 64).to(F16).cuda(), torch.randn(50, 1, 64).to(F16).cuda()
    for bad in ([1, 50], [0, 30, 20, 50], [0, 51], [-1, 50], [0, 60, 50]):
        p = prompt.Packing(torch.tensor(bad, dtype=torch.int32).cuda(), 50)
        leaf = q.clone().requires_grad_()
        o, lse = prompt.prompt_attention(leaf, k, k, p, return_lse=True)
        (gq,) = torch.autograd.grad(o, leaf, q)
        assert not bool(o.any()) and bool((lse == -math.inf).all()) and not bool(gq.any())
        with pytest.raises(RuntimeError, match="offsets"):
            p.check()
    for good in ([0], [0, 0], [0, 50], [0, 0, 10, 10]):
        prompt.Packing(torch.tensor(good, dtype=torch.int32).cuda(), 50).check()


def test_nothing():
    p = prompt.Packing(torch.tensor([0, 0], dtype=torch.int32).cuda(), 0)
    q = torch.zeros(0, 2, 64, dtype=F16, device="cuda").requires_grad_()
    o = prompt.prompt_attention(q, q[:, :1], q[:, :1], p)
    assert o.shape == (0, 2, 64)
    (g,) = torch.autograd.grad(o.sum(), q)
    assert g.shape == q.shape


def test_in_a_graph_that_follows_the_offsets():
    """Replays with other offsets and inputs, the program's own calls between."""
    c = Case([300, 90, 110], 4, 2, 128, BF16, 12)
    n = c.packing.tokens
    offsets = torch.tensor(c.offsets, dtype=torch.int32).cuda()
    leaves = [t.clone().requires_grad_() for t in (c.q, c.k, c.v)]

    def step():
        p = prompt.Packing(offsets, n)
        o, lse = prompt.prompt_attention(*leaves, p, return_lse=True)
        return [o.detach(), lse, *torch.autograd.grad(o, leaves, c.go)]

    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        got = step()
    torch.cuda.current_stream().wait_stream(s)
    assert all(torch.equal(a, b) for a, b in zip(got, c.run()))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step()
    for cuts in (c.offsets, [0, 10, 400, 512], [0, 512, 512, 512], c.offsets):
        offsets.copy_(torch.tensor(cuts, dtype=torch.int32))
        with torch.no_grad():
            leaves[0].mul_(-1)
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, step()))


def test_two_calls_at_once():
    a, b = Case([900, 100], 8, 2, 64, BF16), Case([500, 400, 7], 8, 2, 64, BF16, seed=3)
    want = a.run(), b.run()
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    for _ in range(3):
        got = []
        for s, c in zip(streams, (a, b)):
            s.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(s):
                got.append(c.run())
        for s in streams:
            torch.cuda.current_stream().wait_stream(s)
        torch.cuda.synchronize()
        for g, w in zip(got, want):
            assert all(torch.equal(x, y) for x, y in zip(g, w))


def test_offsets_past_32_bits():
    """More than 2^31 queries: the last sequences, beside a batch of their own."""
    lengths, heads, kv, d = [300] * 1800 + [100, 260], 32, 2, 128
    n = sum(lengths)
    assert n * heads * d > 2**31
    last = sum(lengths[-3:])
    g = torch.Generator(device="cuda").manual_seed(0)
    q = torch.empty(n, heads, d, dtype=BF16, device="cuda")
    for i in range(0, n, 65536):
        q[i:i + 65536].normal_(generator=g)
    k, v = (torch.randn(n, kv, d, generator=g, device="cuda").to(BF16) for _ in range(2))
    p = prompt.Packing(torch.tensor(offsets_of(lengths), dtype=torch.int32).cuda(), n)
    leaves = [t.requires_grad_() for t in (q, k, v)]
    o, lse = prompt.prompt_attention(*leaves, p, return_lse=True)
    got = [o.detach(), lse, *torch.autograd.grad(o, leaves, q.detach())]
    small = prompt.Packing(torch.tensor(offsets_of(lengths[-3:]), dtype=torch.int32).cuda(), last)
    leaves = [t.detach()[-last:].clone().requires_grad_() for t in (q, k, v)]
    ref, tol = packed_attention(*(t.detach() for t in leaves), offsets_of(lengths[-3:]), d ** -0.5, leaves[0].detach())
    for y, r, e in zip(got, ref, tol):
        within(y[-last:], r, e)
    del small
