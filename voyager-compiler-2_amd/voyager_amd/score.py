"""Scores of given tokens under a model's logits, forward and backward.

:func:`token_scores` reads logits once and gives each row's log probability of
its token, the entropy, and the best alternatives: what evaluating a text,
distilling from it or training on it takes of a vocabulary's logits, without
a tensor of probabilities.  ``speculative.verify`` is the choice among drafted
tokens by such probabilities.  Nothing synchronises and every launch goes on
torch's current stream.
"""

import struct
from typing import NamedTuple, Optional

import torch

from ._lib import check, dtype_code, load, no_tangents, once, ptr, stream_on

MAX_TOP = 64
MAX_VOCAB = 1 << 20
#: ``vh_score_desc``
SCORE = struct.Struct("@QqQqqQQQQQQQQQii")
#: ``vh_score_batched_desc`` after its ``vh_score_desc``
BATCHED = struct.Struct("@qq")
_work = {}  # bytes of workspace, by a call's sizes


class Scores(NamedTuple):
    """Of each row, in float32 with natural logarithms: its token's
    ``logprob``, the ``entropy``, and of the ``top`` largest entries, of equal
    ones the first, ``top_logprob`` and ``top_token`` (int64) ``[..., top]``;
    None where ``top`` is 0."""

    logprob: torch.Tensor
    entropy: torch.Tensor
    top_logprob: Optional[torch.Tensor]
    top_token: Optional[torch.Tensor]


def token_scores(logits: torch.Tensor, tokens: torch.Tensor, top: int = 0) -> Scores:
    """Scores of ``tokens [...]`` (int64) under ``logits [..., vocab]``
    (bfloat16, float16 or float32; at most 2^20 entries, fewer than 2^23 rows),
    and the ``top`` best alternatives, at most 64.  Rows with dense entries, at
    one distance or in batches of one distance (``logits[:, :-1]``), are read in
    place; others are copied.

    A negative token pads: its row's results are 0, its alternatives -1, and it
    has no gradient.  A token past the vocabulary, which the host does not
    read, has the log probability NaN, and a gradient of NaN.  Entries of -inf
    are tokens that cannot come; a row of nothing else, or with +inf or NaN, has
    no probabilities: NaN.  Sums are float32.  Differentiable once in the
    logits, through ``logprob``, ``entropy`` and ``top_logprob``."""
    if logits.dim() < 1 or logits.shape[:-1] != tokens.shape:
        raise ValueError(f"token_scores: tokens {list(tokens.shape)} for logits {list(logits.shape)}")
    if logits.dtype not in (torch.bfloat16, torch.float16, torch.float32):
        raise TypeError(f"token_scores: logits must be bfloat16, float16 or float32 (got {logits.dtype})")
    if tokens.dtype is not torch.int64 or tokens.device != logits.device:
        raise ValueError(f"token_scores: tokens must be int64 on {logits.device} (got {tokens.dtype} on {tokens.device})")
    vocab = logits.shape[-1]
    if not 1 <= vocab <= MAX_VOCAB:
        raise ValueError(f"token_scores: a vocabulary of 1 to {MAX_VOCAB} (got {vocab})")
    if not 0 <= top <= min(MAX_TOP, vocab):
        raise ValueError(f"token_scores: 0 to {min(MAX_TOP, vocab)} alternatives (got {top})")
    no_tangents("token_scores", logits)
    t = tokens.reshape(-1)
    if torch.is_grad_enabled() and logits.requires_grad:
        out = _Scores.apply(logits, t, top)
    else:
        out = _scores(logits, t, top, False)[:4 if top else 2]
    shape = tokens.shape
    if len(shape) != 1:
        out = [y.view(shape + y.shape[1:]) for y in out]
    return Scores(*out) if top else Scores(*out, None, None)


def _rows(x):
    """``x [..., vocab]``, or a copy of it, and how its rows lie: their distance, the
    rows of a batch, and the batches' distance."""
    vocab = x.shape[-1]
    if x.is_contiguous():
        return x, vocab, 1 << 31, 0
    if x.stride(-1) == 1 or vocab == 1:
        dims = []  # sizes and strides, of which the inner ones go on where the outer ones' next is
        for n, st in zip(x.shape[:-1], x.stride()):
            if n == 1:
                continue
            if dims and dims[-1][1] == n * st:
                dims[-1] = dims[-1][0] * n, st
            else:
                dims.append((n, st))
        if len(dims) <= 1:
            return x, dims[0][1] if dims else 0, 1 << 31, 0
        if len(dims) == 2:
            return x, dims[1][1], dims[1][0], dims[0][1]
    return x.contiguous(), vocab, 1 << 31, 0


def _scores(x, tokens, top, train):
    (x, step, *batch), tokens = _rows(x), tokens.contiguous()
    rows, vocab = tokens.shape[0], x.shape[-1]
    dev = x.device
    f = dict(dtype=torch.float32, device=dev)
    logprob, entropy = torch.empty(rows, **f), torch.empty(rows, **f)
    stats = torch.empty(rows, 2, **f) if train else None
    best = torch.empty(rows, top, **f) if top else None
    index = torch.empty(rows, top, dtype=torch.int64, device=dev) if top else None
    d = SCORE.pack(x.data_ptr(), step, tokens.data_ptr(), rows, vocab, logprob.data_ptr(), entropy.data_ptr(),
                   ptr(stats) or 0, ptr(best) or 0, ptr(index) or 0, 0, 0, 0, 0, dtype_code(x.dtype), top) + BATCHED.pack(*batch)
    lib = load()
    sizes = (rows, vocab, x.dtype, top)
    need = _work.get(sizes)
    if need is None:
        need = lib.vh_score_workspace_bytes(d)
        if need >= 0:  # or the call says what is wrong
            if len(_work) >= 4096:
                _work.clear()
            _work[sizes] = need
    work = torch.empty(need, dtype=torch.uint8, device=dev) if need > 0 else None
    st = lib.vh_score_batched(d, ptr(work), max(need, 0), stream_on(dev))
    if st:
        check(st, "vh_score_batched")
    return logprob, entropy, best, index, stats


class _Scores(torch.autograd.Function):
    """Keeps the logits and two numbers a row; the probabilities are formed
    again from them."""

    @staticmethod
    def forward(ctx, x, tokens, top):
        logprob, entropy, best, index, stats = _scores(x, tokens, top, True)
        ctx.set_materialize_grads(False)
        ctx.save_for_backward(x, tokens, entropy, stats, index)
        ctx.top = top
        if not top:
            return logprob, entropy
        ctx.mark_non_differentiable(index)
        return logprob, entropy, best, index

    @staticmethod
    def backward(ctx, g_logprob, g_entropy, g_best=None, _=None):
        once("token_scores")
        if g_logprob is None and g_entropy is None and g_best is None:
            return None, None, None
        x, tokens, entropy, stats, index = ctx.saved_tensors
        (x, step, *batch), tokens = _rows(x), tokens.contiguous()
        g = [None if t is None else t.contiguous() for t in (g_logprob, g_entropy, g_best)]
        grad = torch.empty(x.shape, dtype=x.dtype, device=x.device)
        d = SCORE.pack(x.data_ptr(), step, tokens.data_ptr(), tokens.shape[0], x.shape[-1], 0, entropy.data_ptr(), stats.data_ptr(),
                       0, ptr(index) or 0, *(ptr(t) or 0 for t in g), grad.data_ptr(), dtype_code(x.dtype),
                       ctx.top) + BATCHED.pack(*batch)
        st = load().vh_score_batched_backward(d, stream_on(x.device))
        if st:
            check(st, "vh_score_batched_backward")
        return grad, None, None
