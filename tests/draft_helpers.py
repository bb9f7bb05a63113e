"""Plain forms, in float64 on the CPU, of the operators of a step with drafted
tokens: rotary positions, the quantized paged cache, tree attention and the
choice among drafted tokens."""

import math

import torch

HALF = {torch.bfloat16: 2.0**-8, torch.float16: 2.0**-11, torch.float32: 2.0**-24}  # half a step, relative
MOST = {"fp8_e4m3": 448.0, "int8": 127.0}


# ---------------------------------------------------------------- rotary
def turned(x, positions, freq, factor, rotary, interleaved, back=False):
    """Each pair of ``x [batch, tokens, heads, dim]`` as a complex number,
    times factor * exp(i angle)."""
    angle = positions.double()[..., None] * freq
    turn = torch.polar(torch.full_like(angle, factor), -angle if back else angle)[:, :, None]
    y = x.double().clone()
    part = y[..., :rotary]
    if interleaved:
        z = torch.complex(part[..., 0::2], part[..., 1::2]) * turn
        y[..., :rotary] = torch.stack((z.real, z.imag), -1).flatten(-2)
    else:
        z = torch.complex(part[..., : rotary // 2], part[..., rotary // 2:]) * turn
        y[..., :rotary] = torch.cat((z.real, z.imag), -1)
    return y


def turn_tolerance(x, ref, factor, rotary, interleaved):
    """Half a step of the result, and in float32 of each product: the fraction
    of a turn (2^-26 turns: 1.6 half steps of the angle), sine and cosine
    (within 4 half steps), the factor, two products and a sum."""
    m = torch.zeros_like(x, dtype=torch.float64)
    part = x.double()[..., :rotary].abs()
    if interleaved:
        s = part[..., 0::2] + part[..., 1::2]
        m[..., :rotary] = torch.stack((s, s), -1).flatten(-2)
    else:
        s = part[..., : rotary // 2] + part[..., rotary // 2:]
        m[..., :rotary] = torch.cat((s, s), -1)
    return HALF[x.dtype] * ref.abs() + 10 * 2.0**-24 * factor * m + 1e-30


# ----------------------------------------------------------------- cache
def quantized(x, fmt):
    """``(codes as float32, scales)`` by the cache's definition, in float32."""
    most = torch.tensor(MOST[fmt])
    amax = x.float().abs().amax(-1, keepdim=True).clamp(min=2.0**-100)
    y = x.float() * (most / amax)
    codes = y.round() if fmt == "int8" else y.clamp(-448, 448).to(torch.float8_e4m3fn).float()
    return codes, amax / most


def held(x, fmt):
    """What a row reads back as, before its rounding to 16 bits (float32)."""
    if fmt is None:
        return x.float()
    codes, scale = quantized(x, fmt)
    bad = ~torch.isfinite(x.float()).all(-1, keepdim=True)
    return torch.where(bad, math.nan, codes * scale)


# ------------------------------------------------------------- attention
def ancestors(parents):
    """[batch, nodes, nodes] truth values; a node that pads sees nothing."""
    b, t = parents.shape
    see = torch.zeros(b, t, t, dtype=torch.bool)
    for i in range(b):
        for n in range(t):
            way, m = [n], n
            while m > 0 and 0 <= int(parents[i, m]) < m:
                m = int(parents[i, m])
                way.append(m)
            if m == 0:
                see[i, n, way] = True
    return see


def attention(q, k, v, context, see, scale):
    """``q [b, t, heads, d]`` over ``k, v [b, positions, kv, d]`` (float64):
    output, lse, and for the tolerance sum p |v| and the largest sum |q k|."""
    b, t, heads, d = q.shape
    group = heads // k.shape[2]
    o = torch.zeros(b, t, heads, d, dtype=torch.float64)
    lse = torch.full((b, t, heads), -math.inf, dtype=torch.float64)
    mag, dot = torch.zeros_like(o), torch.zeros_like(lse)
    for i in range(b):
        ctx = int(context[i])
        for n in range(t):
            keys = list(range(ctx)) + [ctx + m for m in range(t) if see[i, n, m]]
            if not keys:
                continue
            for h in range(heads):
                kk, vv = k[i, keys, h // group], v[i, keys, h // group]
                s = kk @ q[i, n, h].double() * scale
                p = torch.softmax(s, 0)
                o[i, n, h], lse[i, n, h] = p @ vv, torch.logsumexp(s, 0)
                mag[i, n, h] = p @ vv.abs()
                dot[i, n, h] = (kk.abs() @ q[i, n, h].double().abs()).max() * scale
    return o, lse, mag, dot


def attention_tolerance(dtype, fmt, d, keys, ref, mag, dot, vmax):
    """``(of o, of lse)``.  Scores: d exact products added in float32 and two
    more roundings; the exponential 2^-22; probabilities rounded to float16
    once, or in two parts (2^-22 of float16, 2^-16 of bfloat16); sums of
    `keys` terms in float32; probabilities under float16's least, 2^-24 of the
    largest value each; half a step of the result."""
    score = (d + 4) * 2.0**-24 * dot
    part = 2.0**-16 if fmt is None and dtype == torch.bfloat16 else 2.0**-22 if dtype == torch.float16 else 2.0**-11
    rel = part + 2.0**-21 + keys * 2.0**-24
    o = HALF[dtype] * ref.abs() * (1 + 2.0**-6) + (2 * score[..., None] + rel) * mag + keys * 2.0**-24 * vmax
    return o, score + 2.0**-21 + keys * 2.0**-24 + 2.0**-22 * 16


# ---------------------------------------------------------------- verify
def verify(target, parents, tokens, u, r, draft=None):
    """One sequence at a time, as the definition reads (lists of ints)."""
    target, parents, tokens = target.double(), parents.tolist(), tokens.tolist()
    u, r = u.double().tolist(), r.double().tolist()
    b, t, vocab = target.shape
    out = []
    for i in range(b):
        now, path, told = 0, [0], []
        while True:
            rest, mass, found = target[i, now].clone(), 1.0, None
            q = None if draft is None else draft[i, now].double()
            for n in [n for n in range(now + 1, t) if parents[i][n] == now]:
                x = tokens[i][n]
                ok = 0 <= x < vocab
                if ok and u[i][n] * mass * (1.0 if q is None else float(q[x])) < float(rest[x]):
                    found = n
                    break
                if q is None:
                    if ok:
                        mass = max(mass - float(rest[x]), 0.0)
                        rest[x] = 0.0
                else:
                    less = (rest - mass * q).clamp(min=0)
                    if float(less.sum()) > 0:
                        rest, mass = less, float(less.sum())
            if found is None:
                break
            path.append(found)
            told.append(tokens[i][found])
            now = found
        total = rest.cumsum(0)
        hit = (total > r[i] * total[-1]).nonzero()
        told.append(int(hit[0]) if len(hit) else vocab - 1)
        pad = [-1] * (t - len(path))
        out.append((told + pad, path + pad, len(path)))
    return ([o[0] for o in out], [o[1] for o in out], [o[2] for o in out])
