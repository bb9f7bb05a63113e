"""Tree attention in float64 on the GPU, long contexts too, with what a row's
error may be by what the row sees: keys that it does not see have no part in
its tolerance."""

import math

import torch

from draft_helpers import HALF, MOST, ancestors
from voyager_amd import paged, speculative


def parents_of(b, t, seed):
    g = torch.Generator().manual_seed(seed)
    n = torch.arange(t).expand(b, t)
    return torch.where(n == 0, -1, (torch.rand(b, t, generator=g) * n).long()).int()


def ways(parents):
    """``ancestors`` of many nodes: [batch, nodes, nodes] truth values."""
    b, t = parents.shape
    if t <= 16:
        return ancestors(parents)
    up = parents.long()
    see = torch.zeros(b, t, t, dtype=torch.bool)
    rows = torch.arange(b)
    for n in range(t):  # parents come first
        p = up[:, n]
        ok = (p >= 0) & (p < n) & see[rows, p.clamp(min=0), p.clamp(min=0)] if n else torch.ones(b, dtype=torch.bool)
        if n:
            see[:, n] = see[rows, p.clamp(min=0)] & ok[:, None]
        see[:, n, n] = ok
    return see


class Case:
    """A cache whose pages lie in any order, filled with ``k`` and ``v [b,
    positions, kv, d]``, and its queries."""

    def __init__(self, b, t, heads, kv, d, fmt, dtype, page, contexts, seed=0, spread=1.0, parents="random"):
        g = torch.Generator().manual_seed(seed)
        per = -(-(max(contexts) + t) // page) + 1
        pages = b * per + 3
        self.b, self.t, self.heads, self.kv, self.d, self.fmt, self.dtype, self.page = b, t, heads, kv, d, fmt, dtype, page
        table = torch.randperm(pages, generator=g)[: b * per].reshape(b, per)
        self.table = table.int().cuda()
        self.cache = paged.PagedCache(pages, page, kv, d, fmt=fmt, dtype=dtype)
        self.slots = (table[:, :, None] * page + torch.arange(page)).reshape(b, per * page).cuda()
        self.k, self.v = ((torch.randn(b, per * page, kv, d, generator=g) * torch.exp(
            spread * torch.randn(b, per * page, kv, 1, generator=g))).to(dtype).cuda() for _ in range(2))
        self.q = torch.randn(b, t, heads, d, generator=g).to(dtype).cuda()
        self.context = torch.tensor(contexts, dtype=torch.int32).cuda()
        self.parents = parents_of(b, t, seed + 1) if isinstance(parents, str) else parents
        self.tree = None if self.parents is None else speculative.Tree(self.parents.cuda())
        self.see = torch.ones(b, t, t).tril().bool() if self.parents is None else ways(self.parents)
        self.scale = d ** -0.5
        self.fill()

    def fill(self):
        self.cache.write(self.k.flatten(0, 1), self.v.flatten(0, 1), self.slots.flatten())

    def run(self, workgroups=0):
        """``workgroups`` as the descriptor has it: how many the keys are shared out to."""
        if workgroups == 0:
            return speculative.tree_attention(self.q, self.cache, self.table, self.context, self.tree, scale=self.scale,
                                              return_lse=True)
        from voyager_amd import _lib

        lib, q = _lib.load(), self.q.contiguous()
        o = torch.empty_like(q)
        lse = torch.empty(q.shape[:3], dtype=torch.float32, device="cuda")
        sb, st, sh, _ = q.stride()
        d = bytes(self.cache.c) + speculative.TREE.pack(
            q.data_ptr(), sb, st, sh, self.table.data_ptr(), self.table.stride(0), self.context.data_ptr(),
            0 if self.tree is None else self.tree.masks.data_ptr(), o.data_ptr(), lse.data_ptr(), self.scale,
            _lib.dtype_code(self.dtype), self.b, self.t, self.heads, self.table.shape[1], workgroups)
        need = lib.vh_tree_attention_workspace_bytes(d)
        work = torch.empty(max(need, 16), dtype=torch.uint8, device="cuda")
        _lib.check(lib.vh_tree_attention(d, work.data_ptr(), need, _lib.stream_on(q.device)), "vh_tree_attention")
        return o, lse

    def held(self):
        """What the cache holds, ``[b, positions, kv, d]`` in float64, and each value row's largest magnitude."""
        out = []
        for codes, scales in ((self.cache.k, self.cache.k_scale), (self.cache.v, self.cache.v_scale)):
            c = (codes.double() if self.fmt is None else codes.double() - 128 if self.fmt == "int8" else
                 codes.view(torch.float8_e4m3fn).double())
            c = c if scales is None else c * scales.double()[..., None]
            out.append(c.transpose(1, 2).flatten(0, 1)[self.slots])
        most = out[1].abs().amax(-1) if self.fmt is None else (
            self.cache.v_scale.double().transpose(1, 2).flatten(0, 1)[self.slots] * MOST[self.fmt])
        return out[0], out[1], most

    def exact(self, gone=None, floor=2.0**-34):
        """``(o, lse, tolerance of o, tolerance of lse)``; ``gone [b,
        positions]``: positions that are not there.

        With p a key's share of its row, s its score, dot the largest
        scale * sum |q| |k| that the row sees:

        * scores: d products summed in float32, and six more roundings: (d + 6)
          2^-24 dot, in the numerator and in the sum;
        * the exponential within 2^-22, twice; p times its scale, in a unit:
          2^-23; p in two 16-bit parts: 2^-22 in float16, 2^-16 in bfloat16;
        * sums: one addition a step of 32 keys, 32 products in it, 64 to join
          waves and splits, in units of 2^-24;
        * float16 parts: half of its least value, 2^-25, where the largest
          p * scale of the row lies at 2^9 or more (8-bit caches), or the
          largest p (float16): keys times ``floor``, 2^-34, of the largest
          p * amax, or of the largest value seen;
        * half a step of the result, which has a least size.
        """
        b, t, heads, d = self.q.shape
        group = heads // self.kv
        k, v, amax = self.held()
        o = torch.zeros(b, t, heads, d, dtype=torch.float64, device="cuda")
        lse = torch.full((b, t, heads), -math.inf, dtype=torch.float64, device="cuda")
        tol, tlse = torch.zeros_like(o), torch.zeros_like(lse)
        part = 2.0**-16 if self.cache.dtype == torch.bfloat16 and self.fmt is None else 2.0**-22
        step = torch.finfo(self.dtype).smallest_normal * torch.finfo(self.dtype).eps
        for i in range(b):
            n = int(self.context[i]) + t
            see = torch.ones(t, n, dtype=torch.bool, device="cuda")
            see[:, n - t:] = self.see[i].cuda()
            see &= self.see[i].diagonal().cuda()[:, None]  # a node that pads sees no context either
            if gone is not None:
                see &= ~gone[i, :n].cuda()
            see = see.repeat_interleave(group, 0)
            some = see.any(-1)
            for h in range(self.kv):
                q = self.q[i, :, h * group:(h + 1) * group].double().reshape(t * group, d)
                kk, vv, am = k[i, :n, h], v[i, :n, h], amax[i, :n, h]
                s = (q @ kk.t() * self.scale).masked_fill(~see, -math.inf)
                m = s.amax(-1, keepdim=True).clamp(min=-1e300)
                p = torch.exp(s - m)
                total = p.sum(-1, keepdim=True).clamp(min=1e-300)
                r = p / total
                mag = r @ vv.abs()
                dot = (q.abs() @ kk.abs().t() * self.scale).masked_fill(~see, 0).amax(-1, keepdim=True)
                if self.fmt is None:
                    least = 0 if self.dtype == torch.bfloat16 else (see * am).amax(-1, keepdim=True) * r.amax(-1, keepdim=True)
                else:
                    least = (r * am).amax(-1, keepdim=True)
                score = (d + 6) * 2.0**-24 * dot
                sums = (32 + n / 32 + 64) * 2.0**-24
                out = r @ vv
                e = ((HALF[self.dtype] * out.abs() * (1 + 2.0**-6)).clamp(min=step / 2) + (2 * score + 2.0**-21 + 2.0**-23 + part + 2 * sums) * mag
                     + n * floor * least)
                at = slice(h * group, (h + 1) * group)
                o[i, :, at] = (out * some[:, None]).reshape(t, group, d)
                tol[i, :, at] = e.reshape(t, group, d)
                full = torch.where(some, (m + total.log())[:, 0], -math.inf)
                lse[i, :, at] = full.reshape(t, group)
                tlse[i, :, at] = (score[:, 0] + 2.0**-21 + sums + 4 * 2.0**-24 * full.abs().clamp(max=1e30)).reshape(t, group)
        return o, lse, tol, tlse

    def agrees(self, got, gone=None, floor=2.0**-34):
        o, lse, tol, tlse = self.exact(gone, floor)
        err = (got[0].double() - o).abs()
        assert bool((err <= tol).all()), f"output: {int((~(err <= tol)).sum())} of {err.numel()} beyond, worst {float((err / tol).max()):.2f}"
        empty = torch.isinf(lse)
        assert torch.equal(got[1] == -math.inf, empty) and bool((got[0][empty] == 0).all())
        e = (got[1].double() - lse).abs()[~empty]
        assert bool((e <= tlse[~empty]).all()), f"lse: worst {float((e / tlse[~empty]).max()):.2f}"
