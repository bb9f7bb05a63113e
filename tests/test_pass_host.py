"""The operators of a pass over packed sequences without a GPU: refusals of
arguments, in Python and at the C entries (which check before they launch),
descriptors and workspace sizes."""

import ctypes
import math
import os
import re

import pytest
import torch

from voyager_amd import _lib, rotary, score

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
    assert _size("vh_score_desc") == score.SCORE.size


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


# ----------------------------------------------------------------- scores
def _score(entry="vh_score", work=P, work_bytes=1 << 40, **kw):
    a = dict(logits=P, logits_st=1000, tokens=P, rows=2, vocab=1000, logprob=P, entropy=P, stats=P, top_logprob=P, top_token=P,
             g_logprob=P, g_entropy=0, g_top=0, grad=P, dtype=_lib.VH_F32, top=3)
    a.update(kw)
    d, lib = score.SCORE.pack(*a.values()), _lib.load()
    if entry == "vh_score":
        return lib.vh_score(d, work, work_bytes, None)
    return lib.vh_score_backward(d, None) if entry == "vh_score_backward" else lib.vh_score_workspace_bytes(d)


@pytest.mark.parametrize("kw", [dict(dtype=_lib.VH_U8), dict(dtype=7), dict(rows=-1), dict(rows=1 << 24), dict(vocab=0),
                                dict(vocab=-5), dict(vocab=(1 << 20) + 1), dict(top=-1), dict(top=65), dict(vocab=2)])
def test_score_entries_refuse(kw):
    assert _score(**kw) == 1 and _lib.load().vh_last_error().startswith(b"vh_score:")
    assert _score("vh_score_backward", **kw) == 1 and _lib.load().vh_last_error().startswith(b"vh_score_backward:")
    assert _score("vh_score_workspace_bytes", **kw) == -1


def test_score_entries_need_their_tensors():
    for kw in (dict(logits=0), dict(tokens=0), dict(logprob=0), dict(entropy=0), dict(stats=0), dict(top_logprob=0),
               dict(top_token=0), dict(vocab=100000, work=None), dict(vocab=100000, work=P + 4), dict(vocab=100000, work_bytes=8)):
        assert _score(**kw) == 1
    for kw in (dict(logits=0), dict(tokens=0), dict(entropy=0), dict(stats=0), dict(grad=0), dict(g_top=P, top_token=0)):
        assert _score("vh_score_backward", **kw) == 1


def test_score_workspace_and_nothing():
    need = lambda **kw: _score("vh_score_workspace_bytes", **kw)
    assert need(rows=0) == 0 and need() == 0  # a row of 1000 is one piece
    assert 0 < need(vocab=100000) < need(vocab=100000, top=64)
    # where rows fill the card, pieces are as long as a workgroup holds
    assert need(rows=4096, vocab=32768, dtype=_lib.VH_BF16) == 0
    assert need(rows=4096, vocab=32769, dtype=_lib.VH_BF16) == 4096 * 2 * (3 * 8 + 12)
    assert _score(rows=0, work=None, work_bytes=0) == 0 and _score("vh_score_backward", rows=0) == 0


def test_score_arguments_refused():
    x, t = torch.zeros(2, 3, 100), torch.zeros(2, 3, dtype=torch.int64)
    with pytest.raises(ValueError, match="tokens"):
        score.token_scores(x, t[0])
    with pytest.raises(ValueError, match="int64"):
        score.token_scores(x, t.int())
    with pytest.raises(TypeError, match="float16 or float32"):
        score.token_scores(x.double(), t)
    with pytest.raises(ValueError, match="vocabulary"):
        score.token_scores(x[..., :0], t)
    with pytest.raises(ValueError, match="vocabulary"):
        score.token_scores(torch.zeros(1).expand((1 << 20) + 1), torch.tensor(0))
    for top in (-1, 65, 101):
        with pytest.raises(ValueError, match="alternatives"):
            score.token_scores(x, t, top=top)
    with pytest.raises(ValueError, match="alternatives"):
        score.token_scores(x[..., :4], t, top=5)
    with pytest.raises(ValueError, match="logits"):
        score.token_scores(torch.tensor(1.0), t)
    with pytest.raises(ValueError, match="cuda"):  # no CPU form
        score.token_scores(x, t)


def test_score_refuses_tangents():
    import torch.autograd.forward_ad as fwAD

    x = torch.zeros(2, 8)
    with fwAD.dual_level():
        with pytest.raises(RuntimeError, match="forward-mode"):
            score.token_scores(fwAD.make_dual(x, x), torch.zeros(2, dtype=torch.int64))
