"""Rotary positions of queries and keys, forward and backward, on the GPU.

:class:`Rotary` holds what a model's configuration fixes -- the frequencies,
scaled for long contexts or not, which channels of a head turn and how they
pair up -- and turns queries and keys by their positions in one launch
(``vh_rope``).  The angle is taken in float64 from the position itself, so no
table bounds the positions and far ones lose nothing; ``decode.rope_tables``
is the bfloat16 table of the MX-int8 decode step, which follows its eager
chain's roundings.  :meth:`Rotary.normed` takes the norms of queries and keys
in the same pass.
"""

import math
import struct
from typing import Dict, Optional, Tuple

import torch

from ._lib import check, dtype_code, load, no_tangents, once, ptr, stream_on

MAX_DIM = 512
#: ``vh_rope_desc``: up to ``inverse``, which a call gives, and the rest, which the embedding does
ROPE = struct.Struct("@QQqqqQQqqqQqqqqiiiii")
_ROPE_REST = struct.Struct("=iiif4xQ")
_NONE = (0, 0, 0, 0, 0, 0)
#: ``vh_norm_rope_desc`` after its ``vh_rope_desc``
NORM = struct.Struct("@QQQqqqQqqqQQif")

_SCALING = {"linear": (), "ntk": (), "bands": ("low", "high", "trained"), "yarn": ("low", "high", "trained")}


def frequencies(rotary_dim: int, theta: float, scaling: Optional[Dict] = None) -> Tuple[torch.Tensor, float]:
    """Radians per position of each pair (float64, on the CPU) and the factor
    of cosine and sine.  With r = ``rotary_dim`` and f_j = theta^(-2j/r):

    * ``None``: f_j;
    * ``linear``: f_j / factor;
    * ``ntk``: f_j of the base theta * factor^(r / (r - 2));
    * ``bands``: f_j where the pair turns more than ``high`` times over the
      ``trained`` length, f_j / factor where fewer than ``low`` times, and
      between them mixed in proportion to its turns;
    * ``yarn``: mixed along the pair's index instead, between the (whole)
      indices that turn ``high`` and ``low`` times, and cosine and sine times
      0.1 ln(factor) + 1.
    """
    j = torch.arange(0, rotary_dim, 2, dtype=torch.float64) / rotary_dim
    f = float(theta) ** -j
    if scaling is None:
        return f, 1.0
    kind = scaling.get("kind")
    if kind not in _SCALING:
        raise ValueError(f"Rotary: unknown scaling {kind!r} (one of {', '.join(sorted(_SCALING))})")
    names = ("kind", "factor") + _SCALING[kind]
    if set(scaling) != set(names):
        raise ValueError(f"Rotary: {kind} scaling takes {', '.join(names)} (got {', '.join(map(str, scaling))})")
    factor = float(scaling["factor"])
    if not (factor >= 1.0 and math.isfinite(factor)):
        raise ValueError(f"Rotary: the scaling factor must be at least 1 (got {factor})")
    if kind == "linear":
        return f / factor, 1.0
    if kind == "ntk":
        if rotary_dim <= 2:
            raise ValueError("Rotary: ntk scaling needs more than one pair")
        return (float(theta) * factor ** (rotary_dim / (rotary_dim - 2))) ** -j, 1.0
    low, high, trained = (float(scaling[n]) for n in ("low", "high", "trained"))
    if not (0 < low < high and trained > 0):
        raise ValueError(f"Rotary: {kind} scaling needs 0 < low < high and a trained length")
    if kind == "bands":
        share = ((trained * f / (2 * math.pi) - low) / (high - low)).clamp(0, 1)
        return f * (share + (1 - share) / factor), 1.0
    first, last = (rotary_dim * math.log(trained / (turns * 2 * math.pi)) / (2 * math.log(theta))
                   for turns in (high, low))
    first, last = max(math.floor(first), 0), min(math.ceil(last), rotary_dim - 1)
    ramp = ((torch.arange(rotary_dim // 2, dtype=torch.float64) - first) / max(last - first, 0.001)).clamp(0, 1)
    return f * (1 - ramp) + f / factor * ramp, 0.1 * math.log(factor) + 1.0


class Rotary:
    """Rotary positions of heads of ``dim`` channels, the first ``rotary_dim``
    of which (default: all) turn, in pairs (j, j + rotary_dim / 2) or, with
    ``interleaved``, (2j, 2j + 1).  ``theta`` is the base of the frequencies,
    ``scaling`` a dict as :func:`frequencies` takes it."""

    def __init__(self, dim: int, theta: float = 10000.0, rotary_dim: Optional[int] = None, interleaved: bool = False,
                 scaling: Optional[Dict] = None, device="cuda"):
        rotary_dim = dim if rotary_dim is None else rotary_dim
        if dim <= 0 or dim % 2 or dim > MAX_DIM:
            raise ValueError(f"Rotary: dim must be even and at most {MAX_DIM} (got {dim})")
        if rotary_dim <= 0 or rotary_dim % 2 or rotary_dim > dim:
            raise ValueError(f"Rotary: rotary_dim must be even and at most dim (got {rotary_dim} of {dim})")
        if not (theta > 1.0 and math.isfinite(theta)):
            raise ValueError(f"Rotary: theta must be over 1 (got {theta})")
        self.dim, self.rotary_dim, self.interleaved = dim, rotary_dim, bool(interleaved)
        f, self.factor = frequencies(rotary_dim, theta, scaling)
        self.turns = (f / (2 * math.pi)).to(device)  # per position: the kernel drops whole turns in float64
        self._checked = self._normed = None

    def __call__(self, q: Optional[torch.Tensor], k: Optional[torch.Tensor], positions: torch.Tensor):
        """``q [batch, tokens, heads, dim]`` and ``k [batch, tokens, kv_heads,
        dim]`` (either may be None) turned by ``positions [batch, tokens]`` or
        ``[tokens]`` (int32 or int64), contiguous, of the inputs' dtype
        (bfloat16, float16 or float32).  Views with dense channels are read in
        place.  Differentiable in q and k, any number of times, in reverse mode."""
        given = (None if q is None else (q.shape, q.dtype, q.device), None if k is None else (k.shape, k.dtype, k.device),
                 positions.shape, positions.dtype, positions.device, self.turns.device)
        if given != self._checked:  # a step's sizes are mostly those of the step before
            self._check(q, k, positions)
            self._checked = given
        no_tangents("Rotary", q, k)
        if torch.is_grad_enabled() and ((q is not None and q.requires_grad) or (k is not None and k.requires_grad)):
            return _Turn.apply(q, k, positions, self, False)
        return self._turn(q, k, positions, False)

    def normed(self, q: Optional[torch.Tensor], k: Optional[torch.Tensor], positions: torch.Tensor,
               q_weight: Optional[torch.Tensor], k_weight: Optional[torch.Tensor], eps: float = 1e-6):
        """``q`` and ``k`` normed a head and then turned, in one pass: each
        head's x becomes ``turn(weight * x * (mean(x^2) + eps) ** -0.5)``,
        rounded once.  ``q_weight`` and ``k_weight [dim]`` (of the values' dtype
        or both float32; None where its tensor is) hold for all heads; the rest
        is as in a call of the embedding.  Squares are summed in float32: a
        head whose sum passes its largest value becomes 0, as one with an
        infinity does but in that channel and the one that it turns with, which
        become NaN.  Differentiable once in q, k and the weights, whose gradients
        are summed in a fixed order: of a few heads in float32, of all in float64."""
        wide = [None if t is None else (t.shape, t.dtype, t.device) for t in (q, k, positions, q_weight, k_weight)]
        given = (*wide, eps, self.turns.device)
        if given != self._normed:
            self._check(q, k, positions)
            self._check_weights(q, k, q_weight, k_weight, eps)
            self._normed = given
        no_tangents("Rotary.normed", q, k, q_weight, k_weight)
        if torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in (q, k, q_weight, k_weight)):
            return _NormTurn.apply(q, k, q_weight, k_weight, positions, self, eps)
        return self._norm_turn(q, k, q_weight, k_weight, positions, eps)

    def _check_weights(self, q, k, q_weight, k_weight, eps) -> None:
        x = q if q is not None else k
        dtypes = {w.dtype for w in (q_weight, k_weight) if w is not None}
        for name, t, w in (("q", q, q_weight), ("k", k, k_weight)):
            if (t is None) != (w is None):
                raise ValueError(f"Rotary.normed: {name}_weight is given where {name} is")
            if w is None:
                continue
            if w.shape != (self.dim,) or w.device != self.turns.device:
                raise ValueError(f"Rotary.normed: {name}_weight must be [{self.dim}] on {self.turns.device} "
                                 f"(got {list(w.shape)} on {w.device})")
            if w.dtype not in (x.dtype, torch.float32) or len(dtypes) > 1:
                raise TypeError(f"Rotary.normed: weights must be float32 or {x.dtype}, of one dtype (got {w.dtype})")
        if not 1e-38 <= eps < math.inf:
            raise ValueError(f"Rotary.normed: eps must be positive (got {eps})")

    def _norm_desc(self, x, qd, kd, positions, q_weight, k_weight, grads, eps) -> bytes:
        batch, tokens, _, _ = x.shape
        ps = positions.stride()
        step = ps[0] if len(ps) == 2 and positions.shape[0] > 1 else 0
        w = q_weight if q_weight is not None else k_weight
        return ROPE.pack(*qd[:5], *kd[:5], positions.data_ptr(), step, ps[-1], batch, tokens, qd[5], kd[5],
                         dtype_code(x.dtype), 64 if positions.dtype is torch.int64 else 32, 0) + _ROPE_REST.pack(
                             self.dim, self.rotary_dim, 1 if self.interleaved else 0, self.factor,
                             self.turns.data_ptr()) + NORM.pack(
                                 ptr(q_weight) or 0, ptr(k_weight) or 0, *grads, dtype_code(w.dtype), eps)

    def _norm_turn(self, q, k, q_weight, k_weight, positions, eps):
        qo = ko = None
        qd = kd = _NONE
        if k is not None:
            k, k_weight = _dense(k), k_weight.contiguous()
            ko = torch.empty_like(k, memory_format=torch.contiguous_format)
            kd = (k.data_ptr(), ko.data_ptr(), *k.stride()[:3], k.shape[2])
        if q is not None:
            q, q_weight = _dense(q), q_weight.contiguous()
            qo = torch.empty_like(q, memory_format=torch.contiguous_format)
            qd = (q.data_ptr(), qo.data_ptr(), *q.stride()[:3], q.shape[2])
        x = q if q is not None else k
        d = self._norm_desc(x, qd, kd, positions, q_weight, k_weight, (0,) * 10, eps)
        st = load().vh_norm_rope(d, stream_on(x.device))
        if st:
            check(st, "vh_norm_rope")
        return qo, ko

    def _norm_turn_back(self, q, k, gq, gk, q_weight, k_weight, positions, eps, wanted):
        """Gradients of q, k and the weights, as far as they are ``wanted``; a
        tensor whose result has no gradient has none either."""
        lib, out = load(), [None] * 4
        qd = kd = _NONE
        grads = [0] * 10
        for i, (t, g, w) in enumerate(((q, gq, q_weight), (k, gk, k_weight))):
            if t is None or g is None:
                continue
            t, g = _dense(t), _dense(g)
            if wanted[i]:
                out[i] = torch.empty_like(t, memory_format=torch.contiguous_format)
            if wanted[2 + i]:
                out[2 + i] = torch.empty_like(w, memory_format=torch.contiguous_format)
                if t.numel() == 0:
                    out[2 + i].zero_()
            d = (t.data_ptr(), ptr(out[i]) or 0, *t.stride()[:3], t.shape[2])
            qd, kd = (d, kd) if i == 0 else (qd, d)
            grads[4 * i:4 * i + 4] = g.data_ptr(), *g.stride()[:3]
            grads[8 + i] = ptr(out[2 + i]) or 0
            x = t
            if i == 0:
                q_weight, q, gq = w.contiguous(), t, g  # named: they live until the launch
            else:
                k_weight, k, gk = w.contiguous(), t, g
        d = self._norm_desc(x, qd, kd, positions, q_weight, k_weight, grads, eps)
        need = lib.vh_norm_rope_workspace_bytes(d) if wanted[2] or wanted[3] else 0
        work = torch.empty(need, dtype=torch.uint8, device=x.device) if need > 0 else None
        st = lib.vh_norm_rope_backward(d, ptr(work), max(need, 0), stream_on(x.device))
        if st:
            check(st, "vh_norm_rope_backward")
        return out

    def _check(self, q, k, positions) -> None:
        x = q if q is not None else k
        if x is None:
            raise ValueError("Rotary: neither queries nor keys given")
        for name, t in (("queries", q), ("keys", k)):
            if t is None:
                continue
            if t.dim() != 4 or t.shape[-1] != self.dim or t.shape[:2] != x.shape[:2]:
                raise ValueError(f"Rotary: {name} must be [batch, tokens, heads, {self.dim}] (got {list(t.shape)})")
            if t.dtype != x.dtype or t.dtype not in (torch.bfloat16, torch.float16, torch.float32):
                raise TypeError(f"Rotary: {name} must be bfloat16, float16 or float32, and of one dtype (got {t.dtype})")
            if t.device != self.turns.device:
                raise ValueError(f"Rotary: {name} are on {t.device}, its frequencies on {self.turns.device}")
        if positions.dtype not in (torch.int32, torch.int64):
            raise TypeError(f"Rotary: positions must be int32 or int64 (got {positions.dtype})")
        if positions.device != self.turns.device:
            raise ValueError(f"Rotary: positions are on {positions.device}, its frequencies on {self.turns.device}")
        if tuple(positions.shape) not in ((x.shape[1],), (x.shape[0], x.shape[1]), (1, x.shape[1])):
            raise ValueError(f"Rotary: positions must be [tokens] or [batch, tokens] (got {list(positions.shape)} for "
                             f"{list(x.shape[:2])})")

    def _turn(self, q, k, positions, inverse: bool):
        qo = ko = None
        qd = kd = _NONE
        x = k
        if k is not None:
            if k.stride(3) != 1:
                k = k.contiguous()
            ko = torch.empty_like(k, memory_format=torch.contiguous_format)
            sb, st, sh, _ = k.stride()
            kd = (k.data_ptr(), ko.data_ptr(), sb, st, sh, k.shape[2])
        if q is not None:
            if q.stride(3) != 1:
                q = q.contiguous()
            qo = torch.empty_like(q, memory_format=torch.contiguous_format)
            sb, st, sh, _ = q.stride()
            qd = (q.data_ptr(), qo.data_ptr(), sb, st, sh, q.shape[2])
            x = q
        batch, tokens, _, _ = x.shape
        ps = positions.stride()
        # one position a token for all sequences: no step from one to the next
        step = ps[0] if len(ps) == 2 and positions.shape[0] > 1 else 0
        # the frequencies' address as it is at the call: a copy of the embedding has its own
        d = ROPE.pack(*qd[:5], *kd[:5], positions.data_ptr(), step, ps[-1], batch, tokens, qd[5], kd[5], dtype_code(x.dtype),
                      64 if positions.dtype is torch.int64 else 32, 1 if inverse else 0) + _ROPE_REST.pack(
                          self.dim, self.rotary_dim, 1 if self.interleaved else 0, self.factor, self.turns.data_ptr())
        st = load().vh_rope(d, stream_on(x.device))
        if st:
            check(st, "vh_rope")
        return qo, ko


class _Turn(torch.autograd.Function):
    """The turn is linear and its transpose is the turn back, so the gradient
    is the operator itself, and its own gradient the turn again."""

    @staticmethod
    def forward(ctx, q, k, positions, rotary, inverse):
        ctx.set_materialize_grads(False)
        ctx.save_for_backward(positions)
        ctx.rotary, ctx.inverse = rotary, inverse
        return rotary._turn(q, k, positions, inverse)

    @staticmethod
    def backward(ctx, gq, gk):
        if not ctx.needs_input_grad[0]:
            gq = None
        if not ctx.needs_input_grad[1]:
            gk = None
        if gq is None and gk is None:
            return None, None, None, None, None
        (positions,) = ctx.saved_tensors
        if torch.is_grad_enabled():  # the gradient's own graph is wanted
            gq, gk = _Turn.apply(gq, gk, positions, ctx.rotary, not ctx.inverse)
        else:
            gq, gk = ctx.rotary._turn(gq, gk, positions, not ctx.inverse)
        return gq, gk, None, None, None


def _dense(t: torch.Tensor) -> torch.Tensor:
    """``t`` with dense channels."""
    return t if t.stride(3) == 1 else t.contiguous()


class _NormTurn(torch.autograd.Function):
    """The norm is recomputed from the inputs, which are read again in any
    case, so nothing else is kept."""

    @staticmethod
    def forward(ctx, q, k, q_weight, k_weight, positions, rotary, eps):
        ctx.set_materialize_grads(False)
        ctx.save_for_backward(q, k, q_weight, k_weight, positions)
        ctx.rotary, ctx.eps = rotary, eps
        return rotary._norm_turn(q, k, q_weight, k_weight, positions, eps)

    @staticmethod
    def backward(ctx, gq, gk):
        once("Rotary.normed")
        if gq is None and gk is None:
            return (None,) * 7
        q, k, q_weight, k_weight, positions = ctx.saved_tensors
        out = ctx.rotary._norm_turn_back(q, k, gq, gk, q_weight, k_weight, positions, ctx.eps, ctx.needs_input_grad[:4])
        return (*out, None, None, None)
