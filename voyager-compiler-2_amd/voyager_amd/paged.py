"""A cache of keys and values in pages, quantized as it is written.

:class:`PagedCache` holds the keys and values of many sequences in pages of a
fixed number of tokens.  A token is written to a *slot* (page * page size +
row); which pages a sequence has, and in what order, is a table the caller
keeps.  Rows are held as 8-bit codes with one float32 scale a head and token
(``fp8_e4m3`` or ``int8``) or in the model's own 16-bit type.  Every launch
goes on torch's current stream and nothing synchronises, so writing, reading
and moving can be captured in a HIP graph; indices out of range are left out
and set a device flag that :meth:`PagedCache.check` reads.
"""

import ctypes
from typing import Optional, Tuple

import torch

from . import _lib
from ._lib import check, dtype_code, load, no_tangents, ptr, stream_on

FORMATS = {"fp8_e4m3": _lib.CACHE_E4M3, "int8": _lib.CACHE_INT8}
MAX_DIM = 512


class CacheFlag:
    """The device int32 the kernels OR ``CACHE_ERR_*`` bits into.  Kernels
    never clear it: :meth:`check` reads and clears it."""

    _WHAT = (
        (_lib.CACHE_ERR_SLOT, "a slot is outside the cache (the token was left out)"),
        (_lib.CACHE_ERR_PAGE, "a page of a table, or a node of a path, is not there (its keys were left out)"),
        (_lib.CACHE_ERR_CONTEXT, "a sequence is longer than its pages (its rows are zero)"),
        (_lib.CACHE_ERR_PARENT, "a node's parent is not before it (the node was taken as padding)"),
    )

    def __init__(self, device):
        self.t = torch.zeros(1, dtype=torch.int32, device=device)

    def check(self, what: str) -> None:
        """Synchronising: raise if a kernel flagged an index since the last
        check, and clear the flag."""
        v = int(self.t.item())
        if v:
            self.t.zero_()
            raise RuntimeError(f"voyager_amd {what}: " + "; ".join(msg for bit, msg in self._WHAT if v & bit))


def _int32(t: torch.Tensor, shape: Tuple[int, ...], device, what: str) -> None:
    if t.shape != shape or t.dtype is not torch.int32 or t.device != device:
        raise ValueError(f"{what} must be int32 {list(shape)} on {device} (got {t.dtype} {list(t.shape)} on {t.device})")


class PagedCache:
    """``pages`` pages of ``page`` tokens for ``kv_heads`` heads of ``dim``
    channels (a multiple of 8).  ``fmt`` is ``"fp8_e4m3"``, ``"int8"`` or None
    (held in ``dtype``, bfloat16 or float16, as rows come and go).

    A row x of a head is held as ``round(x * (most / amax))`` and the float32
    scale ``amax / most``, amax its largest magnitude (at least 2^-100) and
    most the format's largest code (448, 127); a row with an infinity or NaN
    reads back as NaN.  ``k``, ``v``: the codes [pages, kv_heads, page, dim]
    (int8 as code + 128); ``k_scale``, ``v_scale``: [pages, kv_heads, page]."""

    def __init__(self, pages: int, page: int, kv_heads: int, dim: int, fmt: Optional[str] = "fp8_e4m3",
                 dtype: torch.dtype = torch.bfloat16, device="cuda"):
        if fmt is not None and fmt not in FORMATS:
            raise ValueError(f"PagedCache: unknown format {fmt!r} (one of {', '.join(FORMATS)}, or None)")
        if dtype not in (torch.bfloat16, torch.float16):
            raise TypeError(f"PagedCache: dtype must be bfloat16 or float16 (got {dtype})")
        if min(pages, page, kv_heads) <= 0 or pages * page >= 1 << 31:
            raise ValueError(f"PagedCache: needs 1 to 2^31 - 1 slots and heads (got {pages} x {page}, {kv_heads} heads)")
        if dim <= 0 or dim % 8 or dim > MAX_DIM:
            raise ValueError(f"PagedCache: dim must be a multiple of 8, at most {MAX_DIM} (got {dim})")
        self.pages, self.page, self.kv_heads, self.dim = pages, page, kv_heads, dim
        self.fmt, self.dtype = fmt, dtype
        held = torch.uint8 if fmt is not None else dtype
        self.k = torch.zeros(pages, kv_heads, page, dim, dtype=held, device=device)
        self.v = torch.zeros_like(self.k)
        self.k_scale = self.v_scale = None
        if fmt is not None:
            self.k_scale = torch.zeros(pages, kv_heads, page, dtype=torch.float32, device=device)
            self.v_scale = torch.zeros_like(self.k_scale)
        self.flag = CacheFlag(device)
        self.device = self.k.device
        code = FORMATS[fmt] if fmt is not None else _lib.CACHE_F16 if dtype == torch.float16 else _lib.CACHE_BF16
        self.c = _lib.Cache(self.k.data_ptr(), self.v.data_ptr(), ptr(self.k_scale), ptr(self.v_scale),
                            self.flag.t.data_ptr(), pages * page, pages, page, kv_heads, dim, code)
        self._c = ctypes.byref(self.c)
        self._bytes = bytes(self.c)
        self._work = {}  # tree_attention's workspace, by its sizes
        self._dtype_code = dtype_code(dtype)

    def check(self) -> None:
        """Synchronising: raise if an index was out of range since the last check."""
        self.flag.check("PagedCache")

    def _slots(self, slots: torch.Tensor) -> int:
        if slots.dtype is not torch.int64 or slots.dim() != 1 or slots.device != self.device:
            raise ValueError(f"PagedCache: slots must be int64 [tokens] on {self.device} (got {slots.dtype} "
                             f"{list(slots.shape)} on {slots.device})")
        return slots.shape[0]

    def write(self, k: torch.Tensor, v: torch.Tensor, slots: torch.Tensor) -> None:
        """Writes ``k`` and ``v [tokens, kv_heads, dim]`` into ``slots
        [tokens]`` (int64, all different; negative: a token that pads, left
        out).  Views with dense channels are read in place."""
        n = self._slots(slots)
        if (k.requires_grad or v.requires_grad) and torch.is_grad_enabled():
            raise RuntimeError("PagedCache.write: the cache passes no gradient; write under torch.no_grad()")
        no_tangents("PagedCache.write", k, v)
        shape = (n, self.kv_heads, self.dim)
        for name, t in (("k", k), ("v", v)):
            if t.shape != shape or t.dtype is not self.dtype or t.device != self.device:
                raise ValueError(f"PagedCache.write: {name} must be {self.dtype} [{n}, {self.kv_heads}, {self.dim}] on "
                                 f"{self.device} (got {t.dtype} {list(t.shape)} on {t.device})")
        k_st, k_sh, k_sc = k.stride()
        if k_sc != 1:
            k = k.contiguous()
            k_st, k_sh, _ = k.stride()
        v_st, v_sh, v_sc = v.stride()
        if v_sc != 1:
            v = v.contiguous()
            v_st, v_sh, _ = v.stride()
        slots = slots.contiguous()
        st = load().vh_paged_write(self._c, k.data_ptr(), k_st, k_sh, v.data_ptr(), v_st, v_sh, self._dtype_code,
                                   slots.data_ptr(), n, stream_on(self.device))
        if st:
            check(st, "vh_paged_write")

    def read(self, slots: torch.Tensor) -> Tuple[torch.Tensor, torch.Tensor]:
        """``(k, v)``, each ``[tokens, kv_heads, dim]`` of the cache's dtype:
        code * scale, rounded once; zeros where the slot is negative."""
        n = self._slots(slots)
        k = torch.empty(n, self.kv_heads, self.dim, dtype=self.dtype, device=self.device)
        v = torch.empty_like(k)
        slots = slots.contiguous()
        st = load().vh_paged_read(self._c, k.data_ptr(), v.data_ptr(), self._dtype_code, slots.data_ptr(), n,
                                  stream_on(self.device))
        if st:
            check(st, "vh_paged_read")
        return k, v

    def keep(self, table: torch.Tensor, context: torch.Tensor, path: torch.Tensor, count: torch.Tensor) -> None:
        """Moves the rows of a verified tree's kept nodes to the end of their
        sequence: with ``path`` and ``count`` as :func:`speculative.verify`
        returns them, the row at position ``context[b] + path[b, i]`` goes to
        ``context[b] + i``, as it is held.  The sequence is then ``context +
        count`` long."""
        b, nodes = path.shape
        _int32(path, (b, nodes), self.device, "PagedCache.keep: path")
        _int32(context, (b,), self.device, "PagedCache.keep: context")
        _int32(count, (b,), self.device, "PagedCache.keep: count")
        _int32(table, (b, table.shape[-1]), self.device, "PagedCache.keep: table")
        table, path, context, count = (_rows(t) for t in (table, path, context, count))
        st = load().vh_paged_keep(self._c, table.data_ptr(), table.stride(0), table.shape[1], context.data_ptr(),
                                  path.data_ptr(), path.stride(0), count.data_ptr(), b, nodes, stream_on(self.device))
        if st:
            check(st, "vh_paged_keep")


def _rows(t: torch.Tensor) -> torch.Tensor:
    """``t`` with a dense last dimension."""
    return t if t.stride(-1) == 1 else t.contiguous()
