"""Plain forms, in float64, of the operators of a pass over packed sequences:
norms with rotary positions, causal attention, scores of given tokens."""

import math

import torch

from draft_helpers import HALF, turned

U = 2.0**-24  # half a step of float32, relative


# ------------------------------------------------------- norms and positions
def spread(x, rotary, interleaved):
    """|x0| + |x1| of every pair, and |x| of the channels that do not turn."""
    m = x.double().abs().clone()
    part = m[..., :rotary].clone()
    if interleaved:
        s = part[..., 0::2] + part[..., 1::2]
        m[..., :rotary] = torch.stack((s, s), -1).flatten(-2)
    else:
        s = part[..., : rotary // 2] + part[..., rotary // 2:]
        m[..., :rotary] = torch.cat((s, s), -1)
    return m


def norm_turned(x, w, positions, freq, factor, rotary, interleaved, eps):
    """``(y, tolerance)``.  r: dim squares summed (half of that in the root) and
    three roundings; two products; then the turn's 10 roundings as for
    vh_rope; half a step of the result, which has a least size."""
    a, dim = x.double(), x.shape[-1]
    z = a * (a.square().mean(-1, keepdim=True) + eps) ** -0.5 * w.double()
    y = turned(z, positions, freq, factor, rotary, interleaved)
    tol = HALF[x.dtype] * y.abs() + (dim / 2 + 15) * U * factor * spread(z, rotary, interleaved) + least(x.dtype)
    return y, tol


def least(dtype):
    """Half of the least step of a type."""
    f = torch.finfo(dtype)
    return f.smallest_normal * f.eps / 2


def norm_turned_back(x, w, g, positions, freq, factor, rotary, interleaved, eps):
    """``(dx, dw, tolerance of dx, tolerance of dw)`` for the result's gradient
    g: the turn back (10 roundings of a pair's magnitudes), r as above, products
    and a sum of dim terms; for dw a sum over all rows."""
    a, dim = x.double(), x.shape[-1]
    r = (a.square().mean(-1, keepdim=True) + eps) ** -0.5
    z = a * r
    back = turned(g.double(), positions, freq, factor, rotary, interleaved, back=True)
    size = factor * spread(g, rotary, interleaved)
    b, bm = back * w.double(), size * w.double().abs()
    dx = r * (b - z * (b * z).mean(-1, keepdim=True))
    c = (dim + 24) * U
    tol = HALF[x.dtype] * dx.abs() + c * r * (bm + z.abs() * 2 * (bm * z.abs()).mean(-1, keepdim=True)) + least(x.dtype)
    rows = (0, 1, 2)
    dw = (back * z).sum(rows)
    n = x.shape[0] * x.shape[1] * x.shape[2]
    tw = HALF[w.dtype] * dw.abs() + (c + n * U) * (size * z.abs()).sum(rows) + least(w.dtype)
    return dx, dw, tol, tw


def within(got, ref, tol, what=""):
    err = (got.detach().double().cpu() - ref.cpu()).abs()
    ok = (err <= tol.cpu()) | (torch.isnan(ref.cpu()) & torch.isnan(err))
    assert bool(ok.all()), f"{what}: {int((~ok).sum())} of {ok.numel()} beyond, worst {float((err / tol.cpu()).max()):.3g}"


# ----------------------------------------------------------------- scores
def scores(logits, tokens, top, g=None, h=None, t=None):
    """``(logprob, entropy, top_logprob, top_token, grad)`` of rows, from the definition."""
    x = logits.double()
    rows, vocab = x.shape
    z = torch.log_softmax(x, -1)
    p = torch.exp(z)
    pz = torch.where(p == 0, 0.0, p * z)
    entropy = -pz.sum(-1)
    pad, past = tokens < 0, tokens >= vocab
    logprob = torch.where(past, math.nan, z.gather(1, tokens.clamp(0, vocab - 1)[:, None])[:, 0])
    # NaN above all, as a sort has it; of equal values the first
    best = torch.sort(x, dim=-1, descending=True, stable=True).indices[:, :top]
    top_logprob = z.gather(1, best)
    grad = None
    if g is not None:
        g, h, t = g.double(), h.double(), t.double()
        at = torch.zeros_like(x).scatter_add_(1, tokens.clamp(0, vocab - 1)[:, None], g[:, None])
        if top:
            at = at.scatter_add_(1, best, t)
        flat = torch.where(p == 0, 0.0, p * (z + entropy[:, None]))
        grad = at - p * (g + t.sum(-1))[:, None] - h[:, None] * flat
        grad = torch.where(past[:, None], math.nan, grad)
        grad[pad] = 0
    for y in (logprob, entropy, top_logprob):
        y[pad] = 0
    best[pad] = -1
    return logprob, entropy, top_logprob, best, grad


def score_tolerances(logits, ref, g=None, h=None, t=None):
    """Of the results of :func:`scores`.  A power's exponent (x - m) log2(e) is
    two roundings of its size, 2^-23 |d| relative in the power, where powers count
    (|d| below 2^4 and a little), and the constant's 2^-25; the power
    2^-22; sums of at most 64 terms a thread, 64 threads, 8 waves and 64 pieces
    joined: under 150 roundings.  A logarithm: 2^-22 of its size."""
    x = logits.double()
    top = x.masked_fill(~torch.isfinite(x), -1e4).amax(-1)
    rel = (32 + 4 + 150) * U
    far = (x.masked_fill(~torch.isfinite(x), 0) - top[:, None]).abs()
    entropy = ref[1]
    lse = torch.logsumexp(x - top[:, None], -1).nan_to_num(0)
    # log of the sum, and the token's own exponent
    t_log = lambda size: rel + 2.0**-22 * (size.abs() + lse.abs() + 1)
    tol = [t_log(ref[0].nan_to_num(0, neginf=0)), 2 * rel * (1 + entropy.nan_to_num(0)) + 2.0**-21 * (lse.abs() + 1)]
    tol.append(rel + 2.0**-22 * (ref[2].nan_to_num(0, neginf=0).abs() + lse.abs()[:, None] + 1))
    if g is not None:
        p = torch.softmax(x, -1).nan_to_num(0)
        size = p * ((g.double().abs() + t.double().abs().sum(-1))[:, None] * (rel + U * (far + 70))
                    + h.double().abs()[:, None] * (2 * rel + 2.0**-21) * (far + entropy.nan_to_num(0)[:, None] + 1 + far * far * U))
        given = sum(y.double().abs() for y in (g, h)).amax() + t.double().abs().sum(-1).amax()
        tol.append(HALF[logits.dtype] * ref[4].nan_to_num(0).abs() + size * 1.01 + 70 * U * ref[4].nan_to_num(0).abs()
                   + least(logits.dtype) + 1e-37 * given)
    return tol


# ------------------------------------------------------------- attention
def packed_attention(q, k, v, offsets, scale, go=None):
    """Causal attention of packed sequences and its gradients for ``go``, one
    sequence and head at a time, with what their errors may be.

    With dot the largest scale * sum |q| |k| that a row sees, w = its weights:

    * scores: d products summed in float32 and six more roundings; the
      exponential within 2^-22; sums of n terms: (n + 64) 2^-24;
    * a weight is rounded once to the values' type for the second product, and
      goes down to 2^-36 of the largest of its row in float16; weights p (1 + e)
      over their own sum give sum p e (v - o) more: |e| times both magnitudes;
    * gradients of weights: dP and D are d products each, D of a result that
      is known to 2^-17 of itself and otherwise as exactly as the output, and they are
      rounded once, going down to 2^-36 of the largest of their row (key) in float16;
    * half a step of each result, which has a least size.
    """
    n, heads, d = q.shape
    kv, group = k.shape[1], heads // k.shape[1]
    f64 = dict(dtype=torch.float64, device=q.device)
    o, lse = torch.zeros(n, heads, d, **f64), torch.full((n, heads), -math.inf, **f64)
    to, tlse = torch.zeros_like(o), torch.zeros_like(lse)
    gq, tq = torch.zeros_like(o), torch.zeros_like(o)
    gk, gv, tk, tv = (torch.zeros(n, kv, d, **f64) for _ in range(4))
    half, small = HALF[q.dtype], least(q.dtype)
    f16 = 2.0**-36 if q.dtype == torch.float16 else 0.0
    for a, b in zip(offsets, offsets[1:]):
        m = b - a
        if m <= 0:
            continue
        hidden = torch.ones(m, m, dtype=torch.bool, device=q.device).triu(1)
        for h in range(heads):
            g = h // group
            qq, kk, vv = q[a:b, h].double(), k[a:b, g].double(), v[a:b, g].double()
            s = (qq @ kk.t() * scale).masked_fill(hidden, -math.inf)
            p, full = torch.softmax(s, -1), torch.logsumexp(s, -1)
            dot = (qq.abs() @ kk.abs().t() * scale).masked_fill(hidden, 0).amax(-1, keepdim=True)
            score = (d + 6) * U * dot + 2.0**-21
            sums = (m + 64) * U
            x = p @ vv
            mag = p @ vv.abs()
            raw = (half + 2 * score + 2 * sums) * (mag + x.abs()) + m * f16 * vv.abs().amax()
            o[a:b, h], to[a:b, h] = x, half * x.abs() * 1.01 + raw + small
            lse[a:b, h], tlse[a:b, h] = full, score[:, 0] + sums + 2.0**-21 * full.abs()
            if go is None:
                continue
            gg = go[a:b, h].double()
            rel = score + tlse[a:b, h][:, None]  # of a weight
            dp, big = gg @ vv.t(), gg.abs() @ vv.abs().t()
            dd = (gg * x).sum(-1, keepdim=True)
            td = (gg.abs() * (raw + 2.0**-16 * x.abs())).sum(-1, keepdim=True) + d * U * (gg.abs() * x.abs()).sum(-1, keepdim=True)
            ds = p * (dp - dd)
            tds = (p * (rel * (dp - dd).abs() + d * U * big + td)).masked_fill(hidden, 0)
            row = (half + sums) * ds.abs() + tds
            gq[a:b, h] = ds @ kk * scale
            tq[a:b, h] = (row + f16 * ds.abs().amax(-1, keepdim=True).expand(m, m).masked_fill(hidden, 0)) @ kk.abs() * scale
            gk[a:b, g] += ds.t() @ qq * scale
            tk[a:b, g] += (row + f16 * ds.abs().amax(0, keepdim=True).expand(m, m).masked_fill(hidden, 0)).t() @ qq.abs() * scale
            gv[a:b, g] += p.t() @ gg
            tv[a:b, g] += (p * (half + rel + sums) + f16).masked_fill(hidden, 0).t() @ gg.abs()
    for t, ref in ((tq, gq), (tk, gk), (tv, gv)):
        t += half * ref.abs() * 1.01 + heads * U * ref.abs() + small
    return (o, lse, gq, gk, gv), (to, tlse, tq, tk, tv)
