"""The bounds of tree attention's key numbers, at the C entry."""

import pytest

from voyager_amd import _lib, speculative

P = 1 << 20


def _entry(batch, table_pages, page, pages=64):
    c = _lib.Cache(P, P, P, P, P, pages * page, pages, page, 2, 64, _lib.CACHE_E4M3)
    d = bytes(c) + speculative.TREE.pack(P, 256, 256, 64, P, 0, P, 0, P, P, 0.125, _lib.VH_BF16, batch, 3, 4, table_pages, 0)
    lib = _lib.load()
    return lib.vh_tree_attention_workspace_bytes(d), lib.vh_tree_attention(d, None, 0, None)


@pytest.mark.parametrize("batch,table_pages,page,pages", [(257, (1 << 27) - 257, 16, 64), (1 << 18, 1 << 21, 16, 64),
                                                          (300, 15, 1 << 27, 1)])
def test_keys_past_what_is_counted_are_refused(batch, table_pages, page, pages):
    """Pieces of 128 keys of all sequences are counted in 32 bits."""
    assert _entry(batch, table_pages, page, pages) == (-1, 1)
    assert b"too many keys" in _lib.load().vh_last_error()


def test_keys_up_to_what_is_counted_are_not():
    need, rc = _entry(255, (1 << 27) - 257, 16)
    assert need > 0 and rc == 1 and b"workspace" in _lib.load().vh_last_error()
