"""Training and scoring on packed documents with the MI355X kernels: norms of
queries and keys with rotary positions, causal attention of packed sequences,
scores of given tokens.

A small random-weight decoder takes documents of different lengths one after
another, without padding between them.  A step raises the log probability of
each next token, weighted (as advantages weight a sampled answer's), and the
entropy a little; scoring gives each document's log probability and what the
model would have said instead.

``python examples/packed_training.py`` prints a few steps.
"""

import os
import sys

import torch
import torch.nn.functional as F

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
sys.path.insert(0, os.path.join(ROOT, "voyager-compiler-2_amd"))

from voyager_amd import prompt, rotary, score  # noqa: E402


class Model:
    """Pre-norm decoder layers in bfloat16, with a norm of every query and key."""

    def __init__(self, vocab=512, hidden=256, heads=8, kv_heads=2, dim=64, layers=2, seed=0, device="cuda"):
        g = torch.Generator().manual_seed(seed)
        w = lambda *s: (torch.randn(*s, generator=g) * s[0] ** -0.5).bfloat16().to(device).requires_grad_()
        ones = lambda *s: torch.ones(*s, dtype=torch.bfloat16, device=device, requires_grad=True)
        self.heads, self.kv_heads, self.dim = heads, kv_heads, dim
        self.embed = torch.randn(vocab, hidden, generator=g).bfloat16().to(device).requires_grad_()
        self.layers = [dict(qkv=w(hidden, (heads + 2 * kv_heads) * dim), q_norm=ones(dim), k_norm=ones(dim),
                            o=w(heads * dim, hidden), up=w(hidden, 2 * hidden), down=w(2 * hidden, hidden))
                       for _ in range(layers)]
        self.head = w(hidden, vocab)
        self.rotary = rotary.Rotary(dim, theta=1e4, device=device)

    def parameters(self):
        return [self.embed, self.head] + [p for w in self.layers for p in w.values()]

    def __call__(self, tokens, positions, packing):
        """Logits ``[tokens, vocab]`` of packed ``tokens [tokens]``."""
        x = self.embed[tokens]
        n = tokens.shape[0]
        for w in self.layers:
            qkv = (F.rms_norm(x, x.shape[-1:]) @ w["qkv"]).view(1, n, self.heads + 2 * self.kv_heads, self.dim)
            q, k, v = qkv.split((self.heads, self.kv_heads, self.kv_heads), 2)
            q, k = self.rotary.normed(q, k, positions, w["q_norm"], w["k_norm"])
            x = x + prompt.prompt_attention(q[0], k[0], v[0], packing).flatten(1) @ w["o"]
            x = x + F.silu(F.rms_norm(x, x.shape[-1:]) @ w["up"]) @ w["down"]
        return F.rms_norm(x, x.shape[-1:]) @ self.head


def pack(documents, rows, device="cuda"):
    """``(tokens, targets, positions, offsets)`` of ``documents`` (lists of
    tokens) in a batch of ``rows``: a target is the next token of the document,
    -1 where there is none."""
    tokens, targets, positions, offsets = [], [], [], [0]
    for d in documents:
        tokens += d
        targets += d[1:] + [-1]
        positions += range(len(d))
        offsets.append(len(tokens))
    pad = rows - len(tokens)
    tensor = lambda x, fill: torch.tensor(x + [fill] * pad, device=device)
    return tensor(tokens, 0), tensor(targets, -1), tensor(positions, 0), torch.tensor(offsets, dtype=torch.int32, device=device)


def loss_of(model, tokens, targets, positions, packing, weights, entropy=0.01):
    """The mean over targets of -weight * log probability - ``entropy`` * entropy."""
    s = score.token_scores(model(tokens, positions, packing), targets)
    return -(weights * s.logprob + entropy * s.entropy).sum() / (targets >= 0).sum()


@torch.no_grad()
def documents_scores(model, tokens, targets, positions, packing, offsets, top=3):
    """Each document's log probability, and every row's best alternatives."""
    s = score.token_scores(model(tokens, positions, packing), targets, top=top)
    upto = F.pad(s.logprob.double().cumsum(0), (1, 0))
    return upto[offsets[1:].long()] - upto[offsets[:-1].long()], s.top_token


def main(steps=5):
    g = torch.Generator().manual_seed(1)
    documents = [torch.randint(0, 512, (n,), generator=g).tolist() for n in (300, 17, 120, 1, 400)]
    model = Model()
    tokens, targets, positions, offsets = pack(documents, 900)
    packing = prompt.Packing(offsets, 900)
    packing.check()
    weights = torch.ones(900, device="cuda")
    optimizer = torch.optim.SGD(model.parameters(), lr=0.5)
    for step in range(steps):
        optimizer.zero_grad()
        loss = loss_of(model, tokens, targets, positions, packing, weights)
        loss.backward()
        optimizer.step()
        print(f"step {step}: loss {float(loss):.3f}", flush=True)
    told, best = documents_scores(model, tokens, targets, positions, packing, offsets)
    for i, d in enumerate(documents):
        print(f"document {i}: {len(d)} tokens, log probability {float(told[i]):.1f}", flush=True)


if __name__ == "__main__":
    main()
