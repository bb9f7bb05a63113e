"""The example of training on packed documents, and its operators together."""

import os
import sys

import pytest
import torch
import torch.nn.functional as F

pytestmark = pytest.mark.gpu
sys.path.insert(0, os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "examples"))


def _documents(lengths):
    g = torch.Generator().manual_seed(1)
    return [torch.randint(0, 512, (n,), generator=g).tolist() for n in lengths]


def _plain(model, document, weight, entropy):
    """The loss's sum over one document, in float64 with torch's own operators."""
    p = {id(x): x for x in model.parameters()}
    d = {k: x.detach().double().requires_grad_() for k, x in p.items()}
    at = lambda x: d[id(x)]
    tokens = torch.tensor(document, device="cuda")
    n, dim, heads, kv = len(document), model.dim, model.heads, model.kv_heads
    f = 1e4 ** -(torch.arange(0, dim, 2, dtype=torch.float64, device="cuda") / dim)
    angle = (torch.arange(n, device="cuda").double()[:, None] * f)[:, None]

    def turned(x, w):
        x = F.rms_norm(x, (dim,), eps=1e-6) * w
        a, b = x[..., :dim // 2], x[..., dim // 2:]
        return torch.cat((a * angle.cos() - b * angle.sin(), b * angle.cos() + a * angle.sin()), -1)

    x = at(model.embed)[tokens]
    hidden = x.shape[-1]
    for w in model.layers:
        eps = torch.finfo(torch.bfloat16).eps  # as rms_norm of bfloat16 takes it
        qkv = (F.rms_norm(x, (hidden,), eps=eps) @ at(w["qkv"])).view(n, heads + 2 * kv, dim)
        q, k, v = qkv.split((heads, kv, kv), 1)
        q, k = turned(q, at(w["q_norm"])), turned(k, at(w["k_norm"])).repeat_interleave(heads // kv, 1)
        v = v.repeat_interleave(heads // kv, 1)
        z = (q.transpose(0, 1) @ k.transpose(0, 1).transpose(1, 2) * dim ** -0.5)
        z = z.masked_fill(torch.ones(n, n, dtype=torch.bool, device="cuda").triu(1), -torch.inf)
        x = x + (z.softmax(-1) @ v.transpose(0, 1)).transpose(0, 1).flatten(1) @ at(w["o"])
        x = x + F.silu(F.rms_norm(x, (hidden,), eps=eps) @ at(w["up"])) @ at(w["down"])
    logp = (F.rms_norm(x, (hidden,), eps=torch.finfo(torch.bfloat16).eps) @ at(model.head)).log_softmax(-1)
    h = -(logp.exp() * logp).sum(-1)
    told = logp[:-1].gather(1, tokens[1:, None])[:, 0] if n > 1 else logp[:0, 0]
    return -(weight * told.sum() + entropy * h[:-1].sum()), [d[id(x)] for x in model.parameters()], told.sum()


def test_losses_gradients_and_scores():
    """Against each document by itself in float64.  A gradient passes some 24
    results that are rounded to bfloat16, of which each is off by at most 2^-8: 0.1 of its norm."""
    import packed_training as example
    from voyager_amd import prompt

    documents = _documents((60, 1, 17, 130))
    model = example.Model()
    tokens, targets, positions, offsets = example.pack(documents, 220)
    packing = prompt.Packing(offsets, 220)
    packing.check()
    weights = torch.full((220,), 0.7, device="cuda")
    loss = example.loss_of(model, tokens, targets, positions, packing, weights, entropy=0.1)
    got = torch.autograd.grad(loss, model.parameters())
    count = int((targets >= 0).sum())
    total, grads, told = 0.0, None, []
    for d in documents:
        y, leaves, t = _plain(model, d, 0.7, 0.1)
        g = torch.autograd.grad(y, leaves)
        grads = list(g) if grads is None else [a + b for a, b in zip(grads, g)]
        total += float(y.detach())
        told.append(float(t))
    assert abs(float(loss) - total / count) < 0.1 * abs(total / count)
    for a, b in zip(got, grads):
        assert float((a.double() - b / count).norm()) < 0.1 * float(b.norm()) / count
    scores, best = example.documents_scores(model, tokens, targets, positions, packing, offsets)
    assert torch.allclose(scores, torch.tensor(told, dtype=torch.float64, device="cuda"), rtol=0.1, atol=0.1)
    assert best.shape == (220, 3) and bool((best[targets < 0] == -1).all()) and bool((best[targets >= 0] >= 0).all())


def test_a_step_in_a_graph():
    """Forward, backward and update, captured: replays take new documents in the same rows."""
    import packed_training as example
    from voyager_amd import prompt

    batches = [example.pack(_documents(n), 300) for n in ((100, 50, 150), (3, 200, 40), (1, 1, 290))]
    weights = torch.ones(300, device="cuda")

    def step(model, tokens, targets, positions, offsets):
        loss = example.loss_of(model, tokens, targets, positions, prompt.Packing(offsets, 300), weights)
        grads = torch.autograd.grad(loss, model.parameters())
        with torch.no_grad():
            for p, g in zip(model.parameters(), grads):
                p.sub_(g, alpha=0.1)
        return loss.detach()

    model, held = example.Model(layers=1), [t.clone() for t in batches[0]]
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        step(model, *held)
    torch.cuda.current_stream().wait_stream(s)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        loss = step(model, *held)
    start = example.Model(layers=1)
    with torch.no_grad():
        for p, q in zip(model.parameters(), start.parameters()):
            p.copy_(q)
    for batch in batches:
        for t, new in zip(held, batch):
            t.copy_(new)
        graph.replay()
        torch.cuda.synchronize()
        want = step(start, *batch)
        # the embedding's gradient is added up by atomics, in any order: equal but for that
        assert torch.allclose(loss, want, rtol=1e-3)
        for p, q in zip(model.parameters(), start.parameters()):
            assert float((p - q).double().norm()) < 1e-2 * float(q.double().norm())


def test_it_runs(capsys):
    import packed_training as example

    example.main(steps=2)
    assert capsys.readouterr().out.count("document") == 5
