"""The operators of a step with drafted tokens without a GPU: the frequencies
of scaled rotary positions, the refusals of arguments, in Python and at the C
entries (which check before they launch), and workspace sizes."""

import ctypes
import math
import os
import re

import pytest
import torch

from voyager_amd import _lib, paged, rotary, speculative


# ---------------------------------------------------------------- rotary
def test_plain_and_linear_frequencies():
    f, factor = rotary.frequencies(8, 10000.0)
    assert factor == 1.0 and torch.allclose(f, torch.tensor([1.0, 0.1, 0.01, 0.001], dtype=torch.float64), rtol=1e-14)
    g, _ = rotary.frequencies(8, 10000.0, {"kind": "linear", "factor": 4.0})
    assert torch.equal(g, f / 4)


def test_ntk_keeps_the_first_pair_and_divides_the_last():
    f, _ = rotary.frequencies(64, 10000.0)
    g, _ = rotary.frequencies(64, 10000.0, {"kind": "ntk", "factor": 8.0})
    assert g[0] == 1.0
    assert math.isclose(float(f[-1] / g[-1]), 8.0, rel_tol=1e-12)  # the slowest pair as linear scaling has it


@pytest.mark.parametrize("kind", ["bands", "yarn"])
def test_mixed_scalings_end_at_whole_and_divided(kind):
    args = {"kind": kind, "factor": 8.0, "low": 1.0, "high": 4.0, "trained": 8192}
    f, _ = rotary.frequencies(128, 5e5)
    g, factor = rotary.frequencies(128, 5e5, args)
    turns = 8192 * f / (2 * math.pi)
    assert torch.equal(g[0], f[0]) and math.isclose(float(g[-1]), float(f[-1]) / 8, rel_tol=1e-12)
    assert bool(((g <= f * (1 + 1e-12)) & (g >= f / 8 * (1 - 1e-12))).all()) and bool((g.diff() < 0).all())
    if kind == "bands":
        assert factor == 1.0
        assert torch.equal(g[turns >= 4], f[turns >= 4]) and torch.allclose(g[turns <= 1], f[turns <= 1] / 8, rtol=1e-12)
    else:
        assert math.isclose(factor, 0.1 * math.log(8) + 1)


@pytest.mark.parametrize("scaling", [
    {"kind": "other", "factor": 2.0}, {"kind": "linear"}, {"kind": "linear", "factor": 0.5},
    {"kind": "linear", "factor": 2.0, "low": 1.0}, {"kind": "bands", "factor": 2.0},
    {"kind": "bands", "factor": 2.0, "low": 4.0, "high": 1.0, "trained": 100},
    {"kind": "yarn", "factor": 2.0, "low": 1.0, "high": 4.0, "trained": 0}])
def test_scalings_refused(scaling):
    with pytest.raises(ValueError):
        rotary.Rotary(64, scaling=scaling, device="cpu")


@pytest.mark.parametrize("kw", [{"dim": 0}, {"dim": 33}, {"dim": 514}, {"dim": 64, "rotary_dim": 66},
                                {"dim": 64, "rotary_dim": 31}, {"dim": 64, "rotary_dim": 0}, {"dim": 64, "theta": 1.0}])
def test_rotary_shapes_refused(kw):
    with pytest.raises(ValueError):
        rotary.Rotary(device="cpu", **kw)


def test_rotary_arguments_refused():
    r = rotary.Rotary(8, device="cpu")
    x, pos = torch.zeros(2, 3, 4, 8), torch.arange(3)
    with pytest.raises(ValueError, match="neither"):
        r(None, None, pos)
    with pytest.raises(ValueError, match="keys must be"):
        r(x, torch.zeros(2, 2, 4, 8), pos)
    with pytest.raises(ValueError, match="queries must be"):
        r(torch.zeros(2, 3, 4, 6), None, pos)
    with pytest.raises(TypeError, match="float16 or float32"):
        r(x.double(), None, pos)
    with pytest.raises(TypeError, match="one dtype"):
        r(x, x.half(), pos)
    with pytest.raises(TypeError, match="positions"):
        r(x, None, pos.float())
    for bad in (torch.arange(2), torch.zeros(3, 3, dtype=torch.int64), torch.zeros(2, 3, 1, dtype=torch.int64)):
        with pytest.raises(ValueError, match="positions"):
            r(x, None, bad)
    with pytest.raises(ValueError, match="cuda"):  # no CPU form
        r(x, None, pos)


def _rope(**kw):
    a = dict(q=1 << 20, heads=4, dim=64, rotary=64, dtype=_lib.VH_F32, pos=1 << 20, bits=64, turns=1 << 20, batch=1)
    a.update(kw)
    d = rotary.ROPE.pack(a["q"], a["q"], 0, 0, 0, 0, 0, 0, 0, 0, a["pos"], 0, 1, a["batch"], 3, a["heads"], 0, a["dtype"],
                         a["bits"], 0) + rotary._ROPE_REST.pack(a["dim"], a["rotary"], 0, 1.0, a["turns"])
    return _lib.load().vh_rope(d, None)


def test_descriptors_are_as_long_as_the_header_says():
    """The packed descriptors against the structures' sizes: pointers and
    int64 of 8 bytes, int32 and float of 4, each at its own alignment."""
    text = open(os.path.join(os.path.dirname(__file__), "..", "include", "voyager_hip.h")).read()

    def size(name):
        at, most = 0, 8
        for line in re.search(r"typedef struct %s \{(.*?)\} %s;" % (name, name), text, re.S).group(1).split(";"):
            line = re.sub(r"/\*.*?\*/", "", line, flags=re.S).strip()
            if not line:
                continue
            for i in range(line.count(",") + 1):
                if line.startswith("vh_cache "):
                    n, a = ctypes.sizeof(_lib.Cache), 8
                else:
                    n = a = 8 if "*" in line or "int64_t" in line else 4
                at = -(-at // a) * a + n
        return -(-at // most) * most

    assert size("vh_cache") == ctypes.sizeof(_lib.Cache)
    assert size("vh_rope_desc") == rotary.ROPE.size + rotary._ROPE_REST.size
    assert size("vh_tree_desc") == ctypes.sizeof(_lib.Cache) + speculative.TREE.size
    assert size("vh_verify_desc") == speculative.VERIFY.size


@pytest.mark.parametrize("kw", [dict(dtype=_lib.VH_U8), dict(dim=63, rotary=2), dict(dim=514), dict(rotary=66),
                                dict(rotary=0), dict(bits=16), dict(q=0), dict(pos=0), dict(turns=0),
                                dict(batch=-1)])
def test_rope_entry_refuses(kw):
    assert _rope(**kw) == 1
    assert _lib.load().vh_last_error().startswith(b"vh_rope")


def test_rope_entry_of_nothing():
    assert _rope(batch=0) == 0 and _rope(heads=0) == 0


# ----------------------------------------------------------------- cache
@pytest.mark.parametrize("kw", [dict(pages=0), dict(page=0), dict(kv_heads=0), dict(dim=12), dict(dim=520),
                                dict(fmt="int4"), dict(pages=1 << 27, page=16)])
def test_cache_shapes_refused(kw):
    a = dict(pages=2, page=16, kv_heads=2, dim=64)
    a.update(kw)
    with pytest.raises(ValueError):
        paged.PagedCache(device="cpu", **a)
    with pytest.raises(TypeError):
        paged.PagedCache(2, 16, 2, 64, dtype=torch.float32, device="cpu")


def test_cache_arguments_refused():
    c = paged.PagedCache(2, 16, 2, 64, device="cpu")
    k, slots = torch.zeros(3, 2, 64, dtype=torch.bfloat16), torch.arange(3)
    with pytest.raises(ValueError, match="slots"):
        c.write(k, k, slots.int())
    with pytest.raises(ValueError, match="slots"):
        c.read(slots[None])
    for bad in (k.half(), k[:2], k[:, :1], k[..., :32]):
        with pytest.raises(ValueError, match="v must be"):
            c.write(k, bad, slots)
    with pytest.raises(RuntimeError, match="gradient"):
        c.write(k.clone().requires_grad_(), k, slots)
    i = lambda *s: torch.zeros(*s, dtype=torch.int32)
    for args in ((i(2, 4).long(), i(2), i(2, 3), i(2)), (i(2, 4), i(3), i(2, 3), i(2)), (i(2, 4), i(2), i(2, 3), i(1)),
                 (i(1, 4), i(2), i(2, 3), i(2))):
        with pytest.raises(ValueError, match="int32"):
            c.keep(*args)


def _cache(**kw):
    a = dict(k=1 << 20, v=1 << 20, k_scale=1 << 20, v_scale=1 << 20, flag=1 << 20, slots=64, pages=4, page=16, kv_heads=2,
             dim=64, fmt=_lib.CACHE_E4M3)
    a.update(kw)
    return _lib.Cache(**a)


BAD_CACHES = [dict(k=None), dict(v=None), dict(flag=None), dict(k_scale=None), dict(fmt=4), dict(fmt=-1), dict(pages=0),
              dict(page=0), dict(dim=60), dict(dim=520), dict(slots=65), dict(k=(1 << 20) + 8),
              dict(pages=1 << 27, slots=1 << 31)]


@pytest.mark.parametrize("kw", BAD_CACHES)
def test_cache_entries_refuse(kw):
    lib, c = _lib.load(), ctypes.byref(_cache(**kw))
    p = 1 << 20
    assert lib.vh_paged_write(c, p, 0, 0, p, 0, 0, _lib.VH_BF16, p, 1, None) == 1
    assert lib.vh_paged_read(c, p, p, _lib.VH_BF16, p, 1, None) == 1
    assert lib.vh_paged_keep(c, p, 4, 4, p, p, 4, p, 1, 4, None) == 1
    assert lib.vh_last_error().startswith(b"vh_paged_keep")


@pytest.mark.parametrize("fmt,dtype", [(_lib.CACHE_F16, _lib.VH_BF16), (_lib.CACHE_BF16, _lib.VH_F16),
                                       (_lib.CACHE_INT8, _lib.VH_F32)])
def test_cache_entries_refuse_types(fmt, dtype):
    lib, c, p = _lib.load(), ctypes.byref(_cache(fmt=fmt)), 1 << 20
    assert lib.vh_paged_write(c, p, 0, 0, p, 0, 0, dtype, p, 1, None) == 1
    assert lib.vh_paged_read(c, p, p, dtype, p, 1, None) == 1


def test_cache_entries_of_nothing():
    lib, c = _lib.load(), ctypes.byref(_cache())
    assert lib.vh_paged_write(c, None, 0, 0, None, 0, 0, _lib.VH_BF16, None, 0, None) == 0
    assert lib.vh_paged_read(c, None, None, _lib.VH_BF16, None, 0, None) == 0
    assert lib.vh_paged_keep(c, None, 4, 4, None, None, 4, None, 0, 4, None) == 0
    assert lib.vh_paged_write(c, None, 0, 0, None, 0, 0, _lib.VH_BF16, None, 1, None) == 1


# ------------------------------------------------------------- attention
def _desc(**kw):
    p = 1 << 20
    a = dict(cache=_cache(), q=p, q_sb=256, q_st=256, q_sh=64, table=p, table_st=4, context=p, masks=p, o=p, lse=p,
             scale=0.125, dtype=_lib.VH_BF16, batch=2, nodes=3, heads=4, table_pages=4, workgroups=0)
    a.update(kw)
    return bytes(a.pop("cache")) + speculative.TREE.pack(*a.values())


def _attention(work=1 << 20, work_bytes=1 << 40, **kw):
    return _lib.load().vh_tree_attention(_desc(**kw), work, work_bytes, None)


@pytest.mark.parametrize("kw", [
    dict(dtype=_lib.VH_F32), dict(heads=3), dict(heads=0), dict(batch=-1), dict(nodes=-1), dict(nodes=1025),
    dict(scale=0.0), dict(scale=-1.0), dict(scale=math.inf), dict(scale=math.nan), dict(workgroups=-1), dict(q=0),
    dict(context=0), dict(table=0), dict(o=0), dict(o=(1 << 20) + 4), dict(work_bytes=8, table_pages=4096),
    dict(work=None, table_pages=4096), dict(work=(1 << 20) + 4, table_pages=4096),
    dict(cache=_cache(page=8, pages=8)), dict(cache=_cache(page=24, slots=96)), dict(cache=_cache(dim=72)),
    dict(cache=_cache(fmt=_lib.CACHE_F16)), dict(cache=_cache(fmt=_lib.CACHE_BF16), dtype=_lib.VH_F16)])
def test_attention_entry_refuses(kw):
    lib = _lib.load()
    assert _attention(**kw) == 1
    assert lib.vh_last_error().startswith(b"vh_tree_attention")


@pytest.mark.parametrize("kw", BAD_CACHES)
def test_attention_entry_refuses_caches(kw):
    lib = _lib.load()
    d = _desc(cache=_cache(**kw))
    assert _attention(cache=_cache(**kw)) == 1 and lib.vh_tree_attention_workspace_bytes(d) == -1


def test_attention_workspace():
    need = lambda **kw: _lib.load().vh_tree_attention_workspace_bytes(_desc(**kw))
    assert need(batch=0) == 0 and need(nodes=0) == 0
    assert need(table_pages=4) == 0  # 64 positions: one split
    assert need(table_pages=4096, workgroups=1) == 0
    # a long table is split: as many parts as workgroups, and one more a sequence
    assert need(table_pages=4096, workgroups=64) == (64 // 2 + 2) * 2 * 6 * 66 * 4
    # and does not grow with what the table might hold
    assert need(table_pages=4096) == need(table_pages=1 << 20)
    assert need(table_pages=0) == 0


def test_attention_of_nothing():
    assert _attention(batch=0, q=0, work=None, work_bytes=0) == 0


def test_attention_arguments_refused():
    c = paged.PagedCache(4, 16, 2, 64, device="cpu")
    q = torch.zeros(2, 3, 4, 64, dtype=torch.bfloat16)
    i = lambda *s: torch.zeros(*s, dtype=torch.int32)
    good = (i(2, 4), i(2))
    for bad in (q[0], q.half(), q[..., :32]):
        with pytest.raises(ValueError, match="q must be"):
            speculative.tree_attention(bad, c, *good)
    with pytest.raises(ValueError, match="query heads"):
        speculative.tree_attention(q[:, :, :3], c, *good)
    with pytest.raises(ValueError, match="context"):
        speculative.tree_attention(q, c, i(2, 4), i(3))
    with pytest.raises(ValueError, match="table"):
        speculative.tree_attention(q, c, i(3, 4), i(2))
    with pytest.raises(RuntimeError, match="gradient"):
        speculative.tree_attention(q.clone().requires_grad_(), c, *good)


def test_tree_refuses():
    for bad in (torch.zeros(3, dtype=torch.int32), torch.zeros(2, 3), torch.zeros(2, 3, dtype=torch.int32)):
        with pytest.raises(ValueError, match="parents"):
            speculative.Tree(bad)  # the last: not on the GPU
    lib, p = _lib.load(), 1 << 20
    assert lib.vh_tree_masks(p, 1, 1025, p, p, None) == 1 and lib.vh_tree_masks(None, 1, 4, p, p, None) == 1
    assert lib.vh_tree_masks(p, -1, 4, p, p, None) == 1 and lib.vh_tree_masks(None, 0, 4, None, None, None) == 0


# ---------------------------------------------------------------- verify
def _verify(**kw):
    p = 1 << 20
    a = dict(target=p, target_sb=4000, target_sn=1000, draft=0, draft_sb=0, draft_sn=0, parents=p, tokens=p, u=p, r=p,
             batch=2, nodes=4, vocab=1000, told=p, path=p, count=p)
    work, work_bytes = kw.pop("work", p), kw.pop("work_bytes", 1 << 30)
    a.update(kw)
    return _lib.load().vh_verify(speculative.VERIFY.pack(*a.values()), work, work_bytes, None)


@pytest.mark.parametrize("kw", [dict(target=0), dict(parents=0), dict(tokens=0), dict(u=0), dict(r=0),
                                dict(told=0), dict(path=0), dict(count=0), dict(work=None), dict(work_bytes=8),
                                dict(work=(1 << 20) + 4), dict(batch=-1), dict(batch=65536), dict(nodes=0),
                                dict(nodes=1025), dict(vocab=0), dict(vocab=(1 << 22) + 1)])
def test_verify_entry_refuses(kw):
    assert _verify(**kw) == 1
    assert _lib.load().vh_last_error().startswith(b"vh_verify")


def test_verify_of_nothing():
    assert _verify(batch=0) == 0
    need = _lib.load().vh_verify_workspace_bytes
    assert need(0, 1000) == 0 and need(2, 0) == 0 and 0 < need(1, 1) < need(3, 1) < need(3, 5000)
