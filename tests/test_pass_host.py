"""The operators of a pass over packed sequences without a GPU: refusals of
arguments, in Python and at the C entries (which check before they launch),
descriptors and workspace sizes."""

import ctypes
import math
import os
import re

import pytest
import torch

from voyager_amd import _lib, prompt, rotary, score

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
    assert _size("vh_prompt_desc") == prompt.PROMPT.size
    text = open(os.path.join(os.path.dirname(__file__), "..", "include", "voyager_hip.h")).read()
    for name, value in (("VH_PROMPT_SHORT", prompt.SHORT), ("VH_PROMPT_MAX_TOKENS", prompt.MAX_TOKENS + 1),
                        ("VH_SCORE_MAX_TOP", score.MAX_TOP), ("VH_SCORE_MAX_VOCAB", score.MAX_VOCAB)):
        assert int(re.search(rf"#define {name} (\d+)", text).group(1)) == value


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
    for kw in (dict(logits=0), dict(tokens=0), dict(logprob=0), dict(entropy=0), dict(top_logprob=0),
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


# ------------------------------------------------------------- attention
def _prompt(entry="vh_prompt_attention", work=P, work_bytes=1 << 50, **kw):
    a = dict(q=P, q_st=256, q_sh=64, k=P, k_st=128, k_sh=64, v=P, v_st=128, v_sh=64, plan=P, o=P, o_low=P, lse=P, go=P,
             go_st=256, go_sh=64, gq=P, gk=P, gv=P, tokens=100, scale=0.125, dtype=_lib.VH_BF16, heads=4, kv_heads=2, dim=64, sequences=1)
    a.update(kw)
    d, lib = prompt.PROMPT.pack(*a.values()), _lib.load()
    if entry == "vh_prompt_attention":
        return lib.vh_prompt_attention(d, None)
    if entry == "vh_prompt_attention_backward":
        return lib.vh_prompt_attention_backward(d, work, work_bytes, None)
    return lib.vh_prompt_attention_workspace_bytes(d)


BACK = "vh_prompt_attention_backward"


@pytest.mark.parametrize("kw", [
    dict(dtype=_lib.VH_F32), dict(dim=96), dict(dim=0), dict(tokens=-1), dict(tokens=1 << 24), dict(heads=3), dict(heads=0),
    dict(kv_heads=0), dict(heads=-4), dict(sequences=-1), dict(scale=0.0), dict(scale=-1.0), dict(scale=math.nan), dict(scale=math.inf),
    dict(q_st=1 << 23), dict(k_st=1 << 23), dict(v_st=1 << 40), dict(go_st=1 << 23),
    dict(tokens=(1 << 24) - 1, heads=1 << 20, kv_heads=1 << 20)])
def test_prompt_entries_refuse(kw):
    assert _prompt(**kw) == 1 and _lib.load().vh_last_error().startswith(b"vh_prompt_attention:")
    assert _prompt(BACK, **kw) == 1 and _lib.load().vh_last_error().startswith(b"vh_prompt_attention_backward:")
    assert _prompt("bytes", **kw) == -1


@pytest.mark.parametrize("kw", [dict(q=0), dict(k=0), dict(v=0), dict(plan=0), dict(o=0), dict(lse=0), dict(q=P + 8), dict(k=P + 2),
                                dict(v=P + 4), dict(o=P + 8), dict(q_st=260), dict(k_sh=4), dict(v_st=-8)])
def test_prompt_entries_need_aligned_tensors(kw):
    assert _prompt(**kw) == 1 and _prompt(BACK, **kw) == 1


@pytest.mark.parametrize("kw", [dict(go=0), dict(o_low=0, tokens=512), dict(gq=0), dict(gk=0), dict(gv=0), dict(go=P + 8), dict(go_sh=2),
                                dict(gk=P + 8), dict(work=None), dict(work=P + 8), dict(work_bytes=16)])
def test_prompt_backward_needs_its_tensors(kw):
    assert _prompt(BACK, **kw) == 1


def test_prompt_workspace_and_nothing():
    need = lambda **kw: _prompt("bytes", **kw)
    assert need(tokens=0) == 0 and 0 < need() < need(tokens=5000) < need(tokens=5000, heads=8)
    assert need(tokens=1 << 20, heads=8, kv_heads=8) == (1 << 20) * 8 * 8  # more blocks than are cut
    assert _prompt(tokens=0, q=0) == 0 and _prompt(BACK, tokens=0, q=0, work=None, work_bytes=0) == 0


def test_packing_entry_refuses():
    lib = _lib.load()
    assert lib.vh_packing_ints(0) == 0 and lib.vh_packing_ints(129) == 2 * (129 + 2)
    assert lib.vh_packing_ints(-1) == -1 and lib.vh_packing_ints(1 << 24) == -1
    for args in ((None, 1, 10, P, P), (P, 1, 10, None, P), (P, 1, 10, P, None), (P, -1, 10, P, P), (P, 1, -1, P, P),
                 (P, 1, 1 << 24, P, P)):
        assert lib.vh_packing(*args, None) == 1


# Launches of 2^32 threads and more, and offsets that every workgroup reads.
@pytest.mark.parametrize("kw", [dict(tokens=(1 << 24) - 1, heads=64, kv_heads=64), dict(tokens=1, heads=1 << 22, kv_heads=1)])
def test_prompt_launches_have_a_limit(kw):
    assert _prompt(**kw) == 1 and b"too many heads" in _lib.load().vh_last_error()
    assert _prompt(BACK, **kw) == 1 and b"too many heads" in _lib.load().vh_last_error()


def test_packing_sequences_have_a_limit():
    for sequences in (1 << 20, 1 << 31, (1 << 63) - 1):
        assert _lib.load().vh_packing(P, sequences, 10, P, P, None) == 1


def test_score_launches_have_a_limit():
    for entry in ("vh_score", "vh_score_backward"):
        assert _score(entry, rows=1 << 23) == 1 and b"rows" in _lib.load().vh_last_error()
    assert _score(rows=1 << 22, vocab=1 << 17) == 1 and b"such a vocabulary" in _lib.load().vh_last_error()
    assert _score("vh_score_backward", rows=1 << 22, vocab=1 << 17) == 1 and b"such a vocabulary" in _lib.load().vh_last_error()


def test_packing_refuses():
    for bad in (torch.zeros(2, dtype=torch.int32), torch.zeros(2), torch.zeros(2, 2, dtype=torch.int32)):
        with pytest.raises(ValueError, match="offsets"):
            prompt.Packing(bad, 4)  # the first: not on the GPU


def test_prompt_arguments_refused():
    class Plan:  # a packing that was made on a GPU
        tokens, sequences, device, _checked = 6, 1, torch.device("cpu"), None

    q, k = torch.zeros(6, 4, 64, dtype=torch.bfloat16), torch.zeros(6, 2, 64, dtype=torch.bfloat16)
    run = prompt.prompt_attention
    for bad in (q[:5], q[None], q.float(), q[..., :32], torch.zeros(6, 4, 96, dtype=torch.bfloat16)):
        with pytest.raises(ValueError, match="q must be"):
            run(bad, k, k, Plan)
    for bad in (k[:5], k.half(), k[0], torch.zeros(6, 2, 128, dtype=torch.bfloat16)):
        with pytest.raises(ValueError, match="k must be"):
            run(q, bad, k, Plan)
    for bad in (k[:, :1], k.half()):
        with pytest.raises(ValueError, match="v must be"):
            run(q, k, bad, Plan)
    for heads, kv in ((3, 2), (0, 2), (4, 0)):
        with pytest.raises(ValueError, match="query heads"):
            run(torch.zeros(6, heads, 64, dtype=torch.bfloat16), *(torch.zeros(6, kv, 64, dtype=torch.bfloat16),) * 2, Plan)
    with pytest.raises(ValueError, match="cuda"):  # no CPU form
        run(q, k, k, type("Other", (), dict(tokens=6, sequences=1, _checked=None, device=torch.device("cpu"), plan=torch.zeros(1))))
    with pytest.raises(ValueError, match="its packing on"):
        run(q, k, k, type("Other", (), dict(tokens=6, _checked=None, device=torch.device("cuda", 0))))


def test_prompt_refuses_tangents():
    import torch.autograd.forward_ad as fwAD

    class Plan:
        tokens, sequences, device, _checked = 6, 1, torch.device("cpu"), None

    k = torch.zeros(6, 2, 64, dtype=torch.bfloat16)
    with fwAD.dual_level():
        with pytest.raises(RuntimeError, match="forward-mode"):
            prompt.prompt_attention(fwAD.make_dual(k, k), k, k, Plan)
