"""Generation with drafted tokens on the MI355X kernels: rotary positions, a
paged quantized cache, attention of a tree of drafts, their verification.

A small random-weight decoder whose logits lean on a table of bigrams, which
is also the draft: each step proposes a tree (two tokens after the last one,
two after each of them, ...), runs all of it through the model at once, keeps
the path that the target agrees with, and moves its cache rows together.  A
step yields one to ``depth + 1`` tokens; drawn with given random numbers they
follow the target's distribution whatever the draft.

``python examples/drafted_tokens.py`` prints the tokens a step yields.
"""

import os
import sys

import torch
import torch.nn.functional as F

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
sys.path.insert(0, os.path.join(ROOT, "voyager-compiler-2_amd"))

from voyager_amd import paged, rotary, speculative  # noqa: E402


class Model:
    """Pre-norm decoder layers over paged caches, one a layer."""

    def __init__(self, vocab=512, hidden=256, heads=8, kv_heads=2, dim=64, layers=2, fmt="fp8_e4m3", seed=0, device="cuda"):
        g = torch.Generator().manual_seed(seed)
        w = lambda *s: (torch.randn(*s, generator=g) * s[0] ** -0.5).bfloat16().to(device)
        self.heads, self.kv_heads, self.dim, self.fmt, self.device = heads, kv_heads, dim, fmt, device
        self.embed = torch.randn(vocab, hidden, generator=g).bfloat16().to(device)
        self.layers = [dict(qkv=w(hidden, (heads + 2 * kv_heads) * dim), o=w(heads * dim, hidden), up=w(hidden, 2 * hidden),
                            down=w(2 * hidden, hidden)) for _ in range(layers)]
        self.head = w(hidden, vocab)
        self.bigrams = 4 * torch.randn(vocab, vocab, generator=g).to(device)
        self.rotary = rotary.Rotary(dim, theta=1e4, device=device)

    def caches(self, pages, page):
        return [paged.PagedCache(pages, page, self.kv_heads, self.dim, fmt=self.fmt, device=self.device) for _ in self.layers]

    def __call__(self, tokens, positions, caches, table, context, tree=None):
        """Logits ``[batch, nodes, vocab]`` of tokens at cache positions
        ``context + n``; ``positions`` are their places in the text."""
        b, t = tokens.shape
        page = caches[0].page
        at = context[:, None].long() + torch.arange(t, device=tokens.device)
        slots = (table.long().gather(1, at // page) * page + at % page).flatten()
        x = self.embed[tokens]
        for w, cache in zip(self.layers, caches):
            qkv = (F.rms_norm(x, x.shape[-1:]) @ w["qkv"]).view(b, t, self.heads + 2 * self.kv_heads, self.dim)
            q, k, v = qkv.split((self.heads, self.kv_heads, self.kv_heads), 2)
            q, k = self.rotary(q, k, positions)
            cache.write(k.flatten(0, 1), v.flatten(0, 1), slots)
            x = x + speculative.tree_attention(q, cache, table, context, tree).flatten(2) @ w["o"]
            x = x + F.silu(F.rms_norm(x, x.shape[-1:]) @ w["up"]) @ w["down"]
        return (F.rms_norm(x, x.shape[-1:]) @ self.head).float() + self.bigrams[tokens]


def balanced(depth, branch):
    """Parents and depths of a tree that branches evenly, level by level."""
    parents, depths, level = [-1], [0], [0]
    for d in range(1, depth + 1):
        first = len(parents)
        parents += [up for up in level for _ in range(branch)]
        depths += [d] * (len(parents) - first)
        level = range(first, len(parents))
    return parents, depths


@torch.no_grad()
def generate(model, prompt, steps, depth=3, branch=2, temperature=1.0, page=16, seed=0):
    """``steps`` steps from ``prompt [batch, tokens]``: ``(told, count)``, each
    step's tokens ``[steps, batch, nodes]`` (-1 past the end) and how many.
    ``depth`` 0 drafts nothing: one token a step.  ``temperature`` 0 takes the
    target's best token."""
    dev = prompt.device
    b, n = prompt.shape
    parents, depths = balanced(depth, branch)
    t = len(parents)
    per = -(-(n + steps * (depth + 1) + t) // page)
    table = torch.randperm(b * per, generator=torch.Generator().manual_seed(1)).reshape(b, per).int().to(dev)
    caches = model.caches(b * per, page)
    tree = speculative.Tree(torch.tensor(parents, dtype=torch.int32, device=dev).expand(b, t))
    depths = torch.tensor(depths, device=dev)
    context = torch.zeros(b, dtype=torch.int32, device=dev)
    if n > 1:  # the prompt but its last token, which is the first step's root
        model(prompt[:, :-1], torch.arange(n - 1, device=dev), caches, table, context)
        context += n - 1
    last = prompt[:, -1]
    best = model.bigrams.topk(branch, -1).indices
    g = torch.Generator(device=dev).manual_seed(seed)
    told, counts = [], []
    for _ in range(steps):
        tokens = last[:, None]
        level = tokens
        for _ in range(depth):
            level = best[level].flatten(1)
            tokens = torch.cat((tokens, level), 1)
        logits = model(tokens, context[:, None].long() + depths, caches, table, context, tree)
        target = (F.one_hot(logits.argmax(-1), logits.shape[-1]).float() if temperature == 0 else
                  (logits / temperature).softmax(-1))
        u, r = torch.rand(b, t, generator=g, device=dev), torch.rand(b, generator=g, device=dev)
        out, path, count = speculative.verify(target, tokens, tree, u, r)
        for cache in caches:
            cache.keep(table, context, path, count)
        context = context + count
        last = out.gather(1, count[:, None].long() - 1)[:, 0]
        told.append(out)
        counts.append(count)
    for cache in caches:
        cache.check()
    tree.check()
    return torch.stack(told), torch.stack(counts)


def main():
    model = Model()
    prompt = torch.randint(0, 512, (4, 37), generator=torch.Generator().manual_seed(3)).cuda()
    told, count = generate(model, prompt, steps=16)
    for i in range(prompt.shape[0]):
        print(f"sequence {i}: {int(count[:, i].sum())} tokens in 16 steps:", *count[:, i].tolist(), flush=True)


if __name__ == "__main__":
    main()
