"""A step that verifies drafted tokens: a tree of them attends to a sequence's
cache at once, and given random numbers say which are kept.

* :class:`Tree`: the drafted tokens of each sequence as a tree;
* :func:`tree_attention`: attention of its nodes over the paged cache (one
  node, or a chain of prompt tokens, is a tree as well);
* :func:`verify`: the drafted tokens against the target's probabilities.

Kept rows are then moved together by :meth:`paged.PagedCache.keep`.  Nothing
synchronises and every launch goes on torch's current stream.
"""

import struct
from typing import Optional, Tuple

import torch

from . import _lib
from ._lib import check, load, no_tangents, stream_on
from .paged import CacheFlag, PagedCache, _int32, _rows

MAX_NODES = _lib.TREE_MAX_NODES


#: ``vh_tree_desc`` after its cache, and ``vh_verify_desc``
TREE = struct.Struct("@QqqqQqQQQQfiiiiii4x")
VERIFY = struct.Struct("@QqqQqqQQQQqqqQQQ")


class Tree:
    """Trees of tokens, one a sequence.  ``parents [batch, nodes]`` (int32, on
    the GPU): the node each node follows, which comes before it, and -1 for the
    first, the sequence's last kept token.  Another node with a negative parent
    pads its tree: it sees nothing and is never taken, nor is one under it.
    At most 1024 nodes.  Parents on the GPU are not read on the host: a
    node whose parent is not before it is taken as padding, and :meth:`check`
    raises."""

    def __init__(self, parents: torch.Tensor):
        if parents.dim() != 2 or parents.dtype != torch.int32 or not parents.is_cuda:
            raise ValueError(f"Tree: parents must be int32 [batch, nodes] on the GPU (got {parents.dtype} "
                             f"{list(parents.shape)} on {parents.device})")
        self.batch, self.nodes = parents.shape
        if not 1 <= self.nodes <= MAX_NODES:
            raise ValueError(f"Tree: 1 to {MAX_NODES} nodes (got {self.nodes})")
        self.parents = parents.contiguous()
        self.device = parents.device
        self.flag = CacheFlag(parents.device)
        self._checked = None
        #: bit m of word m // 64: node m is on the way from the root to the node (itself included)
        self.masks = torch.empty(self.batch, self.nodes, -(-self.nodes // 64), dtype=torch.int64, device=parents.device)
        st = load().vh_tree_masks(self.parents.data_ptr(), self.batch, self.nodes, self.masks.data_ptr(),
                                  self.flag.t.data_ptr(), stream_on(parents.device))
        check(st, "vh_tree_masks")

    def check(self) -> None:
        """Synchronising: raise if a node's parent is not before it."""
        self.flag.check("Tree")


def tree_attention(q: torch.Tensor, cache: PagedCache, table: torch.Tensor, context: torch.Tensor,
                   tree: Optional[Tree] = None, *, scale: Optional[float] = None, return_lse: bool = False):
    """Attention of ``q [batch, nodes, heads, dim]`` (the cache's dtype) over
    each sequence's ``context [batch]`` (int32) cached positions and its tree's
    nodes, whose keys and values have been written at positions ``context +
    n``; ``table [batch, pages]`` (int32) names a sequence's pages in order and
    has room for both.  A node sees the context, itself and the nodes on its
    way from the root; without a ``tree``, all nodes before it (a prompt, or
    one token).  ``heads`` is a multiple of the cache's.  ``scale`` defaults to
    ``dim ** -0.5``.

    Returns the output, contiguous, of q's dtype, and with ``return_lse`` also
    the logarithm of each row's sum of exponentials (float32 ``[batch, nodes,
    heads]``).  Rows that see nothing give 0 and -inf.  Heads of 64, 128 or 256
    channels, pages of a multiple of 16 tokens.  No gradient: it reads a cache."""
    dev = cache.device
    if q.dim() != 4 or q.shape[3] != cache.dim or q.dtype is not cache.dtype or q.device != dev:
        raise ValueError(f"tree_attention: q must be {cache.dtype} [batch, nodes, heads, {cache.dim}] on {dev} "
                         f"(got {q.dtype} {list(q.shape)} on {q.device})")
    if q.requires_grad and torch.is_grad_enabled():
        raise RuntimeError("tree_attention: passes no gradient; call it under torch.no_grad()")
    no_tangents("tree_attention", q)
    b, t, heads, dim = q.shape
    if heads == 0 or heads % cache.kv_heads:
        raise ValueError(f"tree_attention: {heads} query heads over {cache.kv_heads} of the cache")
    _int32(context, (b,), dev, "tree_attention: context")
    _int32(table, (b, table.shape[-1]), dev, "tree_attention: table")
    masks = 0
    if tree is not None:
        if tree.batch != b or tree.nodes != t or tree.device != dev:
            raise ValueError(f"tree_attention: a tree of [{tree.batch}, {tree.nodes}] on {tree.device} for queries [{b}, {t}]")
        masks = tree.masks.data_ptr()
    sb, st, sh, sc = q.stride()
    if sc != 1:
        q = q.contiguous()
        sb, st, sh, _ = q.stride()
    table, context = _rows(table), _rows(context)
    pages = table.shape[1]
    o = torch.empty_like(q, memory_format=torch.contiguous_format)
    lse = torch.empty(b, t, heads, dtype=torch.float32, device=dev) if return_lse else None
    d = cache._bytes + TREE.pack(q.data_ptr(), sb, st, sh, table.data_ptr(), table.stride(0), context.data_ptr(), masks,
                                 o.data_ptr(), 0 if lse is None else lse.data_ptr(),
                                 dim ** -0.5 if scale is None else scale, cache._dtype_code, b, t, heads, pages, 0)
    lib = load()
    sizes = (b, t, heads, pages)
    need = cache._work.get(sizes)
    if need is None:
        need = lib.vh_tree_attention_workspace_bytes(d)
        if need >= 0:  # or the call says what is wrong
            if len(cache._work) >= 4096:
                cache._work.clear()
            cache._work[sizes] = need
    work = torch.empty(need, dtype=torch.uint8, device=dev) if need > 0 else None
    rc = lib.vh_tree_attention(d, None if work is None else work.data_ptr(), need, stream_on(dev))
    if rc:
        check(rc, "vh_tree_attention")
    return (o, lse) if return_lse else o


def verify(target: torch.Tensor, tokens: torch.Tensor, tree: Tree, u: torch.Tensor, r: torch.Tensor,
           draft: Optional[torch.Tensor] = None) -> Tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """The drafted ``tokens [batch, nodes]`` (int64; the first node's is the
    last kept token and is not read) against ``target [batch, nodes, vocab]``
    (float32), the target's probabilities after each node.

    From the first node on, a node's children are tried in order: child n of
    token x is taken if ``u[n] * mass * draft(x) < rest(x)``, where rest begins
    as the target's row and mass as 1; if not, ``rest = max(rest - mass *
    draft, 0)`` and mass is its sum.  ``draft [batch, nodes, vocab]``: the draft
    model's probabilities after each node, from which its children were sampled,
    each on its own (with replacement: a token may come twice, and the rule
    counts on it);
    None: the children were chosen (a draft's best tokens), so draft(x) is 1 for
    the child's own token and rest loses it.  Where no child is taken, the last
    token is drawn from rest by ``r``: the first index at which its running sum
    passes r times the whole (where chosen children left nothing in it, the
    token taken out last).  The tokens then follow the target's distribution
    for ``u [batch, nodes]`` and ``r [batch]`` uniform in [0, 1) (float32).

    Returns ``told [batch, nodes]`` (int64: the tokens taken, then the last; -1
    after them), ``path [batch, nodes]`` (int32: the first node and those taken;
    -1 after them) and ``count [batch]`` (int32: how many of each)."""
    b, t, dev = tree.batch, tree.nodes, tree.device
    given = tuple(None if x is None else (x.shape, x.dtype, x.device) for x in (target, tokens, u, r, draft))
    if given != tree._checked:  # a step's sizes are mostly those of the step before
        vocab = target.shape[-1] if target.dim() == 3 else 0
        for name, x, shape, dtype in (("target", target, (b, t, vocab), torch.float32),
                                      ("draft", draft, (b, t, vocab), torch.float32),
                                      ("tokens", tokens, (b, t), torch.int64), ("u", u, (b, t), torch.float32),
                                      ("r", r, (b,), torch.float32)):
            if x is not None and (x.shape != shape or x.dtype is not dtype or x.device != dev):
                raise ValueError(f"verify: {name} must be {dtype} {list(shape)} on {dev} (got {x.dtype} {list(x.shape)} on "
                                 f"{x.device})")
        if vocab == 0:
            raise ValueError("verify: an empty vocabulary")
        tree._checked = given
    vocab = target.shape[2]
    target = _rows(target)
    tb, tn, _ = target.stride()
    q, qb, qn = 0, 0, 0
    if draft is not None:
        draft = _rows(draft)
        q, (qb, qn, _) = draft.data_ptr(), draft.stride()
    tokens, u, r = tokens.contiguous(), u.contiguous(), r.contiguous()
    told = torch.empty_like(tokens)
    path = torch.empty_like(tree.parents)
    count = torch.empty_like(r, dtype=torch.int32)
    lib = load()
    need = lib.vh_verify_workspace_bytes(b, vocab)
    work = torch.empty(need, dtype=torch.uint8, device=dev)
    st = lib.vh_verify(VERIFY.pack(target.data_ptr(), tb, tn, q, qb, qn, tree.parents.data_ptr(), tokens.data_ptr(),
                                   u.data_ptr(), r.data_ptr(), b, t, vocab, told.data_ptr(), path.data_ptr(),
                                   count.data_ptr()), work.data_ptr(), need, stream_on(dev))
    if st:
        check(st, "vh_verify")
    return told, path, count
