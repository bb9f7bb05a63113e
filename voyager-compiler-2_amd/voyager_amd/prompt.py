"""Attention over whole prompts, packed one after another, forward and backward.

:class:`Packing` is the plan of a packed batch, made once and used by every
layer; :func:`prompt_attention` is causal attention with grouped heads over it.
A prompt's first pass and a training step take it; ``speculative.tree_attention``
reads the cache that tokens are then generated from.  Nothing synchronises and
every launch goes on torch's current stream, so both can be captured in a HIP
graph, which follows the offsets where the packing is made inside it.
"""

import struct
from typing import Optional

import torch

from ._lib import check, dtype_code, load, no_tangents, once, ptr, stream_on

MAX_TOKENS = (1 << 24) - 1
DIMS = (64, 128, 256)
SHORT = 512  # ``VH_PROMPT_SHORT``: sequences of fewer rows take more care in the backward pass
#: ``vh_prompt_desc``
PROMPT = struct.Struct("@QqqQqqQqqQQQQQqqQQQqfiiiii")


class Packing:
    """Sequences packed into ``tokens`` rows: sequence s is the rows
    ``offsets[s]`` to ``offsets[s + 1]`` (int32 ``[sequences + 1]`` on the GPU,
    from 0 on and not falling; equal ones are a sequence of no rows).  Rows
    behind the last sequence pad the batch.  Offsets are read on the device,
    when the packing is made: where they are not so, all rows pad, and
    :meth:`check` raises.  Empty sequences cost nothing, but where there are few rows
    a launch is shaped, and its sums ordered, by the number of sequences.  Fewer
    than 2^24 tokens, and 2^20 sequences."""

    def __init__(self, offsets: torch.Tensor, tokens: int):
        if offsets.dim() != 1 or offsets.dtype is not torch.int32 or not offsets.is_cuda or offsets.shape[0] < 1:
            raise ValueError(f"Packing: offsets must be int32 [sequences + 1] on the GPU (got {offsets.dtype} "
                             f"{list(offsets.shape)} on {offsets.device})")
        if not 0 <= tokens <= MAX_TOKENS:
            raise ValueError(f"Packing: at most {MAX_TOKENS} tokens (got {tokens})")
        self.tokens, self.sequences, self.device = tokens, offsets.shape[0] - 1, offsets.device
        self._checked = None
        lib = load()
        self.flag = torch.zeros(1, dtype=torch.int32, device=offsets.device)
        #: each row's first key, the row after the last that sees it as a key, and the blocks in order
        self.plan = torch.empty(lib.vh_packing_ints(tokens), dtype=torch.int32, device=offsets.device)
        offsets = offsets.contiguous()
        check(lib.vh_packing(offsets.data_ptr(), self.sequences, tokens, self.plan.data_ptr(), self.flag.data_ptr(),
                             stream_on(offsets.device)), "vh_packing")

    def check(self) -> None:
        """Synchronising: raise if the offsets were not from 0 on, fell, or passed the rows."""
        if int(self.flag.item()):
            raise RuntimeError("voyager_amd Packing: offsets must begin at 0, not fall, and end within the rows (all rows pad)")


def prompt_attention(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, packing: Packing, *, scale: Optional[float] = None,
                     return_lse: bool = False):
    """Causal attention of ``q [tokens, heads, dim]`` over ``k`` and ``v
    [tokens, kv_heads, dim]`` (bfloat16 or float16, heads of 64, 128 or 256
    channels, ``heads`` a multiple of ``kv_heads``): each row sees its
    sequence's rows up to itself.  ``scale`` defaults to ``dim ** -0.5``.  Views
    with dense channels and rows aligned to 16 bytes are read in place.

    Returns the output, contiguous, and with ``return_lse`` also the logarithm
    of each row's sum of exponentials (float32 ``[tokens, heads]``, without a
    gradient).  Rows that pad give 0 and -inf, and have gradients of 0.  What a
    row does not see has no part in it, whatever it holds; a row that sees an
    infinity or NaN may be NaN, and bfloat16 values under 2^-94 may count as 0.
    Scores, weights' sums and results are held in float32; weights, and in the
    backward pass their gradients, are rounded to the values' type for the matrix
    instructions (for sequences of fewer than 512 rows in two parts).  Of a score
    of size 2^n some 2^(n - 22) is not known, nor is as much of its weight.
    Differentiable once in q, k and v; sums are in a fixed order."""
    given = (q.shape, q.dtype, q.device, k.shape, k.dtype, k.device, v.shape, v.dtype, v.device)
    if given != packing._checked:  # a layer's sizes are mostly those of the layer before
        _check(q, k, v, packing)
        packing._checked = given
    no_tangents("prompt_attention", q, k, v)
    scale = q.shape[2] ** -0.5 if scale is None else scale
    if torch.is_grad_enabled() and (q.requires_grad or k.requires_grad or v.requires_grad):
        o, lse = _Attention.apply(q, k, v, packing, scale)
    else:
        o, lse = _forward(q, k, v, packing, scale)[:2]
    return (o, lse) if return_lse else o


def _check(q, k, v, packing) -> None:
    t = packing.tokens
    if q.dim() != 3 or q.shape[0] != t or q.shape[2] not in DIMS or q.dtype not in (torch.bfloat16, torch.float16):
        raise ValueError(f"prompt_attention: q must be bfloat16 or float16 [{t}, heads, 64, 128 or 256] (got {q.dtype} "
                         f"{list(q.shape)})")
    for name, x in (("k", k), ("v", v)):
        if x.dim() != 3 or x.shape[0] != t or x.shape[1:] != k.shape[1:] or x.shape[2] != q.shape[2] or x.dtype is not q.dtype:
            raise ValueError(f"prompt_attention: {name} must be {q.dtype} [{t}, kv_heads, {q.shape[2]}] "
                             f"(got {x.dtype} {list(x.shape)})")
    for name, x in (("q", q), ("k", k), ("v", v)):
        if x.device != packing.device:
            raise ValueError(f"prompt_attention: {name} is on {x.device}, its packing on {packing.device}")
    if k.shape[1] == 0 or q.shape[1] == 0 or q.shape[1] % k.shape[1]:
        raise ValueError(f"prompt_attention: {q.shape[1]} query heads over {k.shape[1]}")


def _rows(t: torch.Tensor) -> torch.Tensor:
    """``t`` with dense channels and its rows aligned to 16 bytes."""
    st, sh, sc = t.stride()
    if sc == 1 and not (st | sh) & 7 and not t.data_ptr() & 15 and st < 1 << 23:
        return t
    return t.clone(memory_format=torch.contiguous_format)


def _desc(q, k, v, packing, o, low, lse, scale, go=None, grads=(0, 0, 0)):
    return PROMPT.pack(q.data_ptr(), *q.stride()[:2], k.data_ptr(), *k.stride()[:2], v.data_ptr(), *v.stride()[:2],
                       packing.plan.data_ptr(), o.data_ptr(), ptr(low) or 0, lse.data_ptr(), ptr(go) or 0,
                       *(go.stride()[:2] if go is not None else (0, 0)), *grads, packing.tokens, scale, dtype_code(q.dtype),
                       q.shape[1], k.shape[1], q.shape[2], packing.sequences)


def _forward(q, k, v, packing, scale, train=False):
    q, k, v = _rows(q), _rows(k), _rows(v)
    o = torch.empty_like(q, memory_format=torch.contiguous_format)
    # what the rounding leaves out: the backward pass takes sums over a long sequence's results, in which it would be seen
    low = torch.empty_like(o, dtype=torch.bfloat16) if train else None
    lse = torch.empty((2 if train else 1, *q.shape[:2]), dtype=torch.float32, device=q.device)  # and what it leaves out
    st = load().vh_prompt_attention(_desc(q, k, v, packing, o, low, lse, scale), stream_on(q.device))
    if st:
        check(st, "vh_prompt_attention")
    return o, lse[0], low, lse


class _Attention(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, v, packing, scale):
        o, lse, low, stats = _forward(q, k, v, packing, scale, train=True)
        ctx.set_materialize_grads(False)
        ctx.mark_non_differentiable(lse)
        ctx.save_for_backward(q, k, v, o, low, stats)
        ctx.packing, ctx.scale = packing, scale
        return o, lse

    @staticmethod
    def backward(ctx, go, _):
        once("prompt_attention")
        if go is None:
            return (None,) * 5
        q, k, v, o, low, stats = ctx.saved_tensors
        q, k, v, go = _rows(q), _rows(k), _rows(v), _rows(go)
        grads = [torch.empty_like(t, memory_format=torch.contiguous_format) for t in (q, k, v)]
        d = _desc(q, k, v, ctx.packing, o, low, stats, ctx.scale, go, [t.data_ptr() for t in grads])
        lib = load()
        need = lib.vh_prompt_attention_workspace_bytes(d)
        work = torch.empty(need, dtype=torch.uint8, device=q.device) if need > 0 else None
        st = lib.vh_prompt_attention_backward(d, ptr(work), max(need, 0), stream_on(q.device))
        if st:
            check(st, "vh_prompt_attention_backward")
        return (*grads, None, None)
