"""The operators of a pass over packed sequences without a GPU: refusals of
arguments, in Python and at the C entries (which check before they launch),
descriptors and workspace sizes."""

import ctypes
import math
import os
import re

import pytest
import torch

from voyager_amd import _lib, rotary

P = 1 << 20


def _size(name):
    """A structure's size as the header says: pointers and int64 of 8 bytes,
    int32 and float of 4, each at its own alignment."""
    text = open(os.path.join(os.path.dirname(__file__), "..", "include", "voyager_hip.h")).read()
    at = 0
    for line in re.search(r"typedef struct %s \{(.*?)\} %s;" % (name, name), text, re.S).group(1).split(";"):
        line = re.sub(r"/\*.*?\*/", "", line, flags=re.S).strip()
        if not line:
            continue
        for _ in range(line.count(",") + 1):
            n = a = 8 if "*" in line or "int64_t" in line else 4
            if line.startswith("vh_"):
                n, a = _size(line.split()[0]), 8
            at = -(-at // a) * a + n
    return -(-at // 8) * 8


def test_descriptors_are_as_long_as_the_header_says():
    rope = rotary.ROPE.size + rotary._ROPE_REST.size
    assert _size("vh_rope_desc") == rope
    assert _size("vh_norm_rope_desc") == rope + rotary.NORM.size


# ------------------------------------------------------- norms and positions
def _norm(entry="vh_norm_rope", work=P, work_bytes=1 << 40, **kw):
    a = dict(q=P, q_out=P, heads=4, k=0, kv_heads=0, dim=64, rotary=64, dtype=_lib.VH_F32, pos=P, bits=64, turns=P, batch=1,
             qw=P, kw=0, gq=P, gk=0, gqw=P, gkw=0, wdtype=_lib.VH_F32, eps=1e-6)
    a.update(kw)
    d = rotary.ROPE.pack(a["q"], a["q_out"], 0, 0, 0, a["k"], a["k"], 0, 0, 0, a["pos"], 0, 1, a["batch"], 3, a["heads"],
                         a["kv_heads"], a["dtype"], a["bits"], 0) + rotary._ROPE_REST.pack(
                             a["dim"], a["rotary"], 0, 1.0, a["turns"]) + rotary.NORM.pack(
                                 a["qw"], a["kw"], a["gq"], 0, 0, 0, a["gk"], 0, 0, 0, a["gqw"], a["gkw"], a["wdtype"], a["eps"])
    lib = _lib.load()
    if entry.endswith("backward"):
        return lib.vh_norm_rope_backward(d, work, work_bytes, None)
    return getattr(lib, entry)(d, *(() if entry.endswith("bytes") else (None,)))


BAD_NORMS = [dict(dtype=_lib.VH_U8), dict(dim=63, rotary=2), dict(dim=514), dict(rotary=66), dict(rotary=0), dict(bits=16),
             dict(batch=-1), dict(heads=-1), dict(wdtype=_lib.VH_BF16), dict(wdtype=_lib.VH_I64), dict(eps=0.0),
             dict(eps=-1.0), dict(eps=math.nan), dict(eps=math.inf), dict(batch=1 << 31), dict(heads=1 << 20)]


@pytest.mark.parametrize("kw", BAD_NORMS)
def test_norm_entries_refuse(kw):
    assert _norm(**kw) == 1 and _lib.load().vh_last_error().startswith(b"vh_norm_rope:")
    assert _norm("vh_norm_rope_backward", **kw) == 1 and _lib.load().vh_last_error().startswith(b"vh_norm_rope_backward:")
    assert _norm("vh_norm_rope_workspace_bytes", **kw) == -1


@pytest.mark.parametrize("kw", [dict(q=0), dict(qw=0), dict(pos=0), dict(turns=0), dict(kv_heads=2), dict(kv_heads=2, k=P)])
def test_norm_entries_refuse_missing_tensors(kw):
    assert _norm(**kw) == 1 and _norm("vh_norm_rope_backward", **kw) == 1


def test_norm_entry_needs_its_results_and_workspace():
    assert _norm(q_out=0) == 1
    for kw in (dict(gq=0), dict(work=None), dict(work=P + 4), dict(work_bytes=8), dict(kv_heads=2, k=P, kw=P)):
        assert _norm("vh_norm_rope_backward", **kw) == 1
    assert _norm("vh_norm_rope_workspace_bytes") >= 2 * 64 * 4


def test_norm_entries_of_nothing():
    assert _norm(batch=0) == 0 and _norm(heads=0, q=0) == 0
    assert _norm("vh_norm_rope_backward", batch=0, work=None, work_bytes=0) == 0
    assert _norm("vh_norm_rope_workspace_bytes", batch=0) == 0


def test_norm_arguments_refused():
    r = rotary.Rotary(8, device="cpu")
    x, pos, w = torch.zeros(2, 3, 4, 8), torch.arange(3), torch.ones(8)
    with pytest.raises(ValueError, match="neither"):
        r.normed(None, None, pos, None, None)
    with pytest.raises(ValueError, match="q_weight is given"):
        r.normed(x, None, pos, None, None)
    with pytest.raises(ValueError, match="k_weight is given"):
        r.normed(x, None, pos, w, w)
    with pytest.raises(ValueError, match="q_weight must be"):
        r.normed(x, None, pos, w[:4], None)
    with pytest.raises(ValueError, match="k_weight must be"):
        r.normed(x, x, pos, w, w[None])
    with pytest.raises(TypeError, match="weights must be"):
        r.normed(x, None, pos, w.half(), None)
    with pytest.raises(TypeError, match="one dtype"):
        r.normed(x.half(), x.half(), pos, w, w.half())
    with pytest.raises(ValueError, match="queries must be"):
        r.normed(x[0], None, pos, w, None)
    for eps in (0.0, -1e-6, math.nan, math.inf):
        with pytest.raises(ValueError, match="eps"):
            r.normed(x, None, pos, w, None, eps=eps)
    with pytest.raises(ValueError, match="cuda"):  # no CPU form
        r.normed(x, None, pos, w, None)


def test_norm_refuses_tangents():
    import torch.autograd.forward_ad as fwAD

    r = rotary.Rotary(8, device="cpu")
    x, w = torch.zeros(2, 3, 4, 8), torch.ones(8)
    with fwAD.dual_level():
        with pytest.raises(RuntimeError, match="forward-mode"):
            r.normed(x, None, torch.arange(3), fwAD.make_dual(w, w), None)
