"""The operators of a pass over whole packed sequences, as cases that can be timed and checked.

A prompt's first pass, the scoring of a given text and the step that trains on
it take three operators, and a case is one of them:

* ``norm_rope``: norms of queries and keys a head, and their rotary positions,
  in one pass (``voyager_amd.rotary``);
* ``attention``: causal attention of packed sequences with grouped heads
  (``voyager_amd.prompt``);
* ``score``: log probabilities of given tokens, with the entropy and the best
  alternatives (``voyager_amd.score``).

With ``train`` the gradients as well.  Sizes are those of ``bench.py``, the
tests and ``operators.py`` (32 query and 8 key heads of 128, contexts of 4096,
vocabularies of 32,000 and 128,000) or generic.
"""

import math
import os
import sys

import torch

own = False

_ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
_PKG = os.path.join(_ROOT, "voyager-compiler-2_amd")
if _PKG not in sys.path:
    sys.path.insert(0, _PKG)

DEV = "cuda"
DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
SIZE = {"bf16": 2, "fp16": 2, "fp32": 4}
THETA = 5e5
EPS = 1e-6


# ------------------------------------------------------------------ the cases
def listed():
    return [
        # one new token of one user: the smallest call
        {"name": "norm_rope_one_token", "op": "norm_rope", "batch": 1, "tokens": 1, "heads": 32, "kv_heads": 8, "dim": 128,
         "rotary": 128, "dtype": "bf16", "interleaved": False, "weights": "bf16", "train": False},
        # a training step's queries and keys
        {"name": "norm_rope_train_4x2048", "op": "norm_rope", "batch": 4, "tokens": 2048, "heads": 32, "kv_heads": 8,
         "dim": 128, "rotary": 128, "dtype": "bf16", "interleaved": False, "weights": "fp32", "train": True},
        # an odd number of tokens in float32, half of each head turned, side by side
        {"name": "norm_rope_part_fp32_5001", "op": "norm_rope", "batch": 1, "tokens": 5001, "heads": 16, "kv_heads": 4,
         "dim": 128, "rotary": 64, "dtype": "fp32", "interleaved": True, "weights": "fp32", "train": True},
        # one short question of one user: latency
        {"name": "attention_33", "op": "attention", "tokens": 33, "sequences": 1, "padded": False, "heads": 32, "kv_heads": 8,
         "dim": 128, "dtype": "bf16", "train": False},
        # a prompt as long as the context
        {"name": "attention_4096", "op": "attention", "tokens": 4096, "sequences": 1, "padded": False, "heads": 32,
         "kv_heads": 8, "dim": 128, "dtype": "bf16", "train": False},
        # many short prompts in one batch that is padded to its size
        {"name": "attention_64_prompts_fp16", "op": "attention", "tokens": 8001, "sequences": 64, "padded": True, "heads": 16,
         "kv_heads": 16, "dim": 64, "dtype": "fp16", "train": False},
        # a training step on documents of different lengths
        {"name": "attention_train_8192", "op": "attention", "tokens": 8192, "sequences": 6, "padded": False, "heads": 32,
         "kv_heads": 8, "dim": 128, "dtype": "bf16", "train": True},
        # the same of a smaller model, ragged, in the other type
        {"name": "attention_train_5001_fp16", "op": "attention", "tokens": 5001, "sequences": 3, "padded": False, "heads": 16,
         "kv_heads": 4, "dim": 64, "dtype": "fp16", "train": True},
        # a sampled token of one user, with five alternatives
        {"name": "score_1x32000_top5", "op": "score", "rows": 1, "vocab": 32000, "dtype": "fp32", "top": 5, "train": False},
        # a step of 32 users with a large vocabulary and twenty alternatives
        {"name": "score_32x128000_top20", "op": "score", "rows": 32, "vocab": 128000, "dtype": "bf16", "top": 20,
         "train": False},
        # a ragged batch of text scored, every token with its best alternative
        {"name": "score_4001x32000_top1", "op": "score", "rows": 4001, "vocab": 32000, "dtype": "fp16", "top": 1,
         "train": False},
        # a training step that raises given tokens' probabilities and the entropy, large vocabulary
        {"name": "score_train_2048x128000", "op": "score", "rows": 2048, "vocab": 128000, "dtype": "bf16", "top": 0,
         "train": True},
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, round(math.exp(rng.uniform(math.log(lo), math.log(hi))))))


def draw(rng):
    op = rng.choice(["norm_rope", "attention", "attention", "score"])
    kv = rng.choice([1, 2, 4, 8])
    heads = kv * rng.choice([1, 2, 3, 4, 7, 8])
    dim = rng.choice([64, 128, 128, 256])
    if op == "norm_rope":
        dtype = rng.choice(["bf16", "fp16", "fp32"])
        batch = rng.choice([1, 1, 2, 3, 8])
        most = 8192 * 40 * 128 // (batch * (heads + kv) * dim * (2 if dtype == "fp32" else 1))
        return {"op": op, "batch": batch, "tokens": _log(rng, 1, max(1, min(5001, most))), "heads": heads, "kv_heads": kv,
                "dim": dim, "rotary": rng.choice([dim, dim, dim // 2, 32]), "dtype": dtype,
                "interleaved": rng.random() < 0.5, "weights": rng.choice([dtype, "fp32"]), "train": rng.random() < 0.5}
    if op == "attention":
        most = min(8192, int(8192 * math.sqrt(32 * 128 / (heads * dim))))
        tokens = _log(rng, 1, most)
        return {"op": op, "tokens": tokens, "sequences": _log(rng, 1, min(64, tokens)), "padded": rng.random() < 0.5,
                "heads": heads, "kv_heads": kv, "dim": dim, "dtype": rng.choice(["bf16", "fp16"]),
                "train": rng.random() < 0.5}
    vocab = _log(rng, 1000, 128000)
    dtype = rng.choice(["bf16", "fp16", "fp32"])
    train = rng.random() < 0.5
    most = 2048 * 128000 // (vocab * (2 if dtype == "fp32" else 1))
    return {"op": op, "rows": _log(rng, 1, min(4001, most)), "vocab": vocab, "dtype": dtype,
            "top": rng.choice([0, 1, 5, _log(rng, 2, 64)]), "train": train}


# ------------------------------------------------------------------- inputs
def _gen(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def _offsets(case, g):
    """Where the sequences begin and end: cut at random places, so that some are short and some may be empty."""
    held = case["tokens"] - (case["tokens"] // 8 if case["padded"] else 0)
    cuts = torch.randint(0, held + 1, (case["sequences"] - 1,), generator=g, device=DEV)
    ends = torch.tensor([0, held], device=DEV)
    return torch.cat((ends, cuts)).sort().values.to(torch.int32)


def prepare(case, seed):
    g = _gen(seed)
    s = {"case": case}
    dt = DTYPES[case["dtype"]]

    def normal(*shape):
        return torch.randn(*shape, generator=g, device=DEV)

    if case["op"] == "score":
        rows, vocab = case["rows"], case["vocab"]
        # logits with a few tokens far above the rest
        x = normal(rows, vocab)
        x += 2.0 * x * (x > 2.0)
        s["logits"] = (x * 1.5).to(dt)
        s["tokens"] = torch.where(torch.rand(rows, generator=g, device=DEV) < 0.7, s["logits"].argmax(-1),
                                  torch.randint(0, vocab, (rows,), generator=g, device=DEV))
        if case["train"]:
            s["gp"], s["gh"] = normal(rows), 0.1 * normal(rows)
            s["gt"] = 0.1 * normal(rows, case["top"])
            if own:
                s["logits"].requires_grad_()
        return s
    heads, kv, dim = case["heads"], case["kv_heads"], case["dim"]
    if case["op"] == "norm_rope":
        shape = (case["batch"], case["tokens"])
        # as a fused projection leaves them: queries, keys and values of a token side by side
        qkv = (normal(*shape, heads + 2 * kv, dim) * torch.exp(0.5 * normal(*shape, heads + 2 * kv, 1))).to(dt)
        s["q"], s["k"] = qkv[:, :, :heads], qkv[:, :, heads:heads + kv]
        wt = DTYPES[case["weights"]]
        s["qw"], s["kw"] = ((1 + 0.2 * normal(dim)).to(wt) for _ in range(2))
        start = torch.randint(0, 100000, (case["batch"], 1), generator=g, device=DEV)
        s["pos"] = start + torch.arange(case["tokens"], device=DEV)
        s["freq"] = THETA ** -(torch.arange(0, case["rotary"], 2, dtype=torch.float64, device=DEV) / case["rotary"])
        if case["train"]:
            s["gq"], s["gk"] = normal(*shape, heads, dim).to(dt), normal(*shape, kv, dim).to(dt)
        if own:
            from voyager_amd import rotary
            s["rotary"] = rotary.Rotary(dim, theta=THETA, rotary_dim=case["rotary"], interleaved=case["interleaved"],
                                        device=DEV)
            if case["train"]:
                for n in ("q", "k", "qw", "kw"):
                    s[n].requires_grad_()
        return s
    tokens = case["tokens"]
    s["offsets"] = _offsets(case, g)
    # queries and keys that some heads match sharply
    s["q"] = (normal(tokens, heads, dim) * torch.exp(0.5 * normal(1, heads, 1))).to(dt)
    kvs = normal(tokens, 2 * kv, dim).to(dt)
    s["k"], s["v"] = kvs[:, :kv], kvs[:, kv:]
    if case["train"]:
        s["go"] = normal(tokens, heads, dim).to(dt)
    if own:
        from voyager_amd import prompt
        s["packing"] = prompt.Packing(s["offsets"], tokens)
        if case["train"]:
            for n in ("q", "k", "v"):
                s[n].requires_grad_()
    return s


# ------------------------------------------------------------------ one pass
def _turned(x, cos, sin, rotary, interleaved):
    if interleaved:
        x0, x1 = x[..., 0:rotary:2], x[..., 1:rotary:2]
        y = torch.stack((x0 * cos - x1 * sin, x1 * cos + x0 * sin), -1).flatten(-2)
    else:
        x0, x1 = x[..., :rotary // 2], x[..., rotary // 2:rotary]
        y = torch.cat((x0 * cos - x1 * sin, x1 * cos + x0 * sin), -1)
    return torch.cat((y, x[..., rotary:]), -1)


def _norm_rope_one(x, w, gy, cos, sin, how):
    a, weight = x.float(), w.float()
    r = torch.rsqrt(a.square().mean(-1, keepdim=True) + EPS)
    unit = a * r
    y = _turned(unit * weight, cos, sin, *how).to(x.dtype)
    if gy is None:
        return [y]
    g = _turned(gy.float(), cos, -sin, *how)
    gu = g * weight
    gx = r * (gu - unit * (gu * unit).mean(-1, keepdim=True))
    return [y, gx.to(x.dtype), (g * unit).double().sum((0, 1, 2)).to(w.dtype)]


def _norm_rope(s):
    c = s["case"]
    if own:
        y = s["rotary"].normed(s["q"], s["k"], s["pos"], s["qw"], s["kw"], eps=EPS)
        if not c["train"]:
            return list(y)
        grads = torch.autograd.grad(y, (s["q"], s["qw"], s["k"], s["kw"]), (s["gq"], s["gk"]))
        return [y[0].detach(), *grads[:2], y[1].detach(), *grads[2:]]
    angle = s["pos"].double()[..., None, None] * s["freq"]
    cos, sin = angle.cos().float(), angle.sin().float()
    how = (c["rotary"], c["interleaved"])
    return (_norm_rope_one(s["q"], s["qw"], s.get("gq"), cos, sin, how)
            + _norm_rope_one(s["k"], s["kw"], s.get("gk"), cos, sin, how))


def _attention(s):
    c = s["case"]
    if own:
        from voyager_amd import prompt
        o, lse = prompt.prompt_attention(s["q"], s["k"], s["v"], s["packing"], return_lse=True)
        if not c["train"]:
            return [o, lse]
        return [o.detach(), lse.detach(), *torch.autograd.grad(o, (s["q"], s["k"], s["v"]), s["go"])]
    n, heads, kv, d = c["tokens"], c["heads"], c["kv_heads"], c["dim"]
    group, scale = heads // kv, 1 / math.sqrt(d)
    at = torch.arange(n, device=DEV)
    # each token's sequence; those behind the last have none
    which = torch.searchsorted(s["offsets"], at.to(torch.int32), right=True)
    hidden = (which[:, None] != which[None, :]) | (at[None, :] > at[:, None]) | (at >= s["offsets"][-1])[:, None]
    q = s["q"].float().reshape(n, kv, group, d).permute(1, 2, 0, 3).reshape(kv, group * n, d)
    k, v = s["k"].float().transpose(0, 1), s["v"].float().transpose(0, 1)
    x = (q @ k.transpose(1, 2) * scale).reshape(kv, group, n, n).masked_fill_(hidden, -math.inf)
    m = x.amax(-1, keepdim=True).clamp(min=torch.finfo(torch.float32).min)
    x = x.sub_(m).exp_()
    total = x.sum(-1, keepdim=True)
    p = x.div_(total.clamp(min=1e-30)).reshape(kv, group * n, n)
    o = p @ v

    def rows(y):
        return y.reshape(kv, group, n, d).permute(2, 0, 1, 3).reshape(n, heads, d)

    out = [rows(o).to(s["q"].dtype), (m + total.log()).reshape(heads, n).t().contiguous()]
    if not c["train"]:
        return out
    go = s["go"].float().reshape(n, kv, group, d).permute(1, 2, 0, 3).reshape(kv, group * n, d)
    gv = p.transpose(1, 2) @ go
    gs = (go @ v.transpose(1, 2)).sub_((go * o).sum(-1, keepdim=True)).mul_(p)
    gq, gk = gs @ k * scale, gs.transpose(1, 2) @ q * scale
    return out + [rows(gq).to(s["q"].dtype), gk.transpose(0, 1).to(s["q"].dtype), gv.transpose(0, 1).to(s["q"].dtype)]


def _score(s):
    c = s["case"]
    if own:
        from voyager_amd import score
        r = score.token_scores(s["logits"], s["tokens"], top=c["top"])
        out = [r.logprob, r.entropy] + ([r.top_logprob, r.top_token] if c["top"] else [])
        if not c["train"]:
            return out
        ends = [r.logprob, r.entropy] + ([r.top_logprob] if c["top"] else [])
        grad = torch.autograd.grad(ends, s["logits"], [s["gp"], s["gh"], s["gt"]][:len(ends)])
        return [x.detach() for x in out] + list(grad)
    x = s["logits"].float()
    y = x - x.amax(-1, keepdim=True)
    e = y.exp()
    total = e.sum(-1, keepdim=True)
    logp = y - total.log()
    p = e / total
    entropy = -(p * logp).sum(-1)
    at = s["tokens"][:, None]
    out = [logp.gather(1, at)[:, 0], entropy]
    if c["top"]:  # a stable sort: of equal values the lowest index first
        best = torch.sort(x, dim=-1, descending=True, stable=True).indices[:, :c["top"]]
        out += [logp.gather(1, best), best]
    if not c["train"]:
        return out
    g = -p * (s["gp"][:, None] + s["gt"].sum(-1, keepdim=True) + s["gh"][:, None] * (logp + entropy[:, None]))
    g.scatter_add_(1, at, s["gp"][:, None])
    if c["top"]:
        g.scatter_add_(1, best, s["gt"])
    return out + [g.to(s["logits"].dtype)]


def run(state):
    return {"norm_rope": _norm_rope, "attention": _attention, "score": _score}[state["case"]["op"]](state)


# -------------------------------------------------------------- what it takes
def work(case):
    size = SIZE[case["dtype"]]
    if case["op"] == "norm_rope":
        values = case["batch"] * case["tokens"] * (case["heads"] + case["kv_heads"]) * case["dim"]
        # x in, y out; and of the gradients dy in, dx out
        return {"bytes": (4 if case["train"] else 2) * values * size + 8 * case["batch"] * case["tokens"],
                "flops": (24 if case["train"] else 7) * values}
    if case["op"] == "attention":
        held = case["tokens"] - (case["tokens"] // 8 if case["padded"] else 0)
        pairs = (2 * held * held / (case["sequences"] + 1) + held) / 2  # the mean over the places of the cuts
        d, heads, kv = case["dim"], case["heads"], case["kv_heads"]
        values = case["tokens"] * d * (2 * heads + 2 * kv)
        return {"bytes": (2 if case["train"] else 1) * values * size + 4 * case["tokens"] * heads,
                "flops": (14 if case["train"] else 4) * pairs * heads * d}
    values = case["rows"] * case["vocab"]
    return {"bytes": (2 if case["train"] else 1) * values * size + case["rows"] * (16 + 12 * case["top"]),
            "flops": (12 if case["train"] else 5) * values}


# --------------------------------------------------------- the values in 64 bits
def exact(case, seed):
    global own
    was, own = own, False
    s = prepare(case, seed)
    own = was
    if case["op"] == "norm_rope":
        half = case["rotary"] // 2
        turn = torch.polar(torch.ones_like(s["pos"].double()[..., None] * s["freq"]),
                           s["pos"].double()[..., None] * s["freq"])[:, :, None]

        def by(x, w):  # pairs as complex numbers
            y = x.clone()
            r = y[..., :case["rotary"]]
            pair = r.unflatten(-1, (half, 2)) if case["interleaved"] else r.unflatten(-1, (2, half)).transpose(-1, -2)
            z = torch.view_as_real(torch.view_as_complex(pair.contiguous()) * w)
            y[..., :case["rotary"]] = z.flatten(-2) if case["interleaved"] else z.transpose(-1, -2).flatten(-2)
            return y

        out = []
        for x, w, gy in ((s["q"], s["qw"], s.get("gq")), (s["k"], s["kw"], s.get("gk"))):
            a, weight = x.double(), w.double()
            n = (a * a).sum(-1, keepdim=True) / case["dim"] + EPS
            out.append(by(a * weight / n.sqrt(), turn))
            if gy is not None:
                g = by(gy.double(), turn.conj())
                b = g * weight
                out.append(b / n.sqrt() - a * (a * b).sum(-1, keepdim=True) / (case["dim"] * n * n.sqrt()))
                out.append((g * a / n.sqrt()).flatten(0, 2).sum(0))
        return out
    if case["op"] == "attention":
        heads, kv, d = case["heads"], case["kv_heads"], case["dim"]
        o = torch.zeros(case["tokens"], heads, d, dtype=torch.float64, device=DEV)
        lse = torch.full((case["tokens"], heads), -math.inf, dtype=torch.float64, device=DEV)
        gq = torch.zeros_like(o)
        gk, gv = (torch.zeros(case["tokens"], kv, d, dtype=torch.float64, device=DEV) for _ in range(2))
        ends = s["offsets"].tolist()
        for a, b in zip(ends, ends[1:]):
            later = torch.ones(b - a, b - a, dtype=torch.bool, device=DEV).triu(1)
            for h in range(heads if b > a else 0):
                g = h * kv // heads
                q, k, v = s["q"][a:b, h].double(), s["k"][a:b, g].double(), s["v"][a:b, g].double()
                z = torch.where(later, -math.inf, q @ k.t() / math.sqrt(d))
                lse[a:b, h] = torch.logsumexp(z, -1)
                p = torch.softmax(z, -1)
                o[a:b, h] = p @ v
                if case["train"]:
                    go = s["go"][a:b, h].double()
                    dp = go @ v.t()
                    ds = p * (dp - (p * dp).sum(-1, keepdim=True)) / math.sqrt(d)
                    gq[a:b, h] = ds @ k
                    gk[a:b, g] += ds.t() @ q
                    gv[a:b, g] += p.t() @ go
        return [o, lse, gq, gk, gv] if case["train"] else [o, lse]
    logprob, entropy, best, alternatives, grad = [], [], [], [], []
    for i in range(0, case["rows"], 256):
        x, t = s["logits"][i:i + 256].double(), s["tokens"][i:i + 256, None]
        z = x - torch.logsumexp(x, -1, keepdim=True)
        p = torch.exp(z)
        h = -(p * z).sum(-1, keepdim=True)
        logprob.append(z.gather(1, t)[:, 0])
        entropy.append(h[:, 0])
        if case["top"]:
            index = torch.sort(x, dim=-1, descending=True, stable=True).indices[:, :case["top"]]
            best.append(index)
            alternatives.append(z.gather(1, index))
        if case["train"]:
            gp, gh = s["gp"][i:i + 256, None].double(), s["gh"][i:i + 256, None].double()
            given = torch.zeros_like(x).scatter_add_(1, t, gp)
            if case["top"]:
                given.scatter_add_(1, index, s["gt"][i:i + 256].double())
            grad.append((given - p * given.sum(-1, keepdim=True) - gh * p * (z + h)).float())
    out = [logprob, entropy] + ([alternatives, best] if case["top"] else []) + ([grad] if case["train"] else [])
    return [torch.cat(x) for x in out]
