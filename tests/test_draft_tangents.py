"""Forward-mode derivatives: the operators of a step with drafted tokens have
none and say so, where they would be taken as zero."""

import pytest
import torch
from torch.autograd import forward_ad

from voyager_amd import paged, rotary, speculative


def _dual(x):
    return forward_ad.make_dual(x, torch.ones_like(x))


@pytest.mark.parametrize("which", ["q", "k", "both"])
@pytest.mark.parametrize("grad", [False, True])
def test_rotary(which, grad):
    r = rotary.Rotary(8, device="cpu")
    q, k = (torch.zeros(1, 2, 3, 8, requires_grad=grad) for _ in range(2))
    with forward_ad.dual_level():
        args = (_dual(q) if which != "k" else q, _dual(k) if which != "q" else k)
        with pytest.raises(RuntimeError, match="Rotary: no forward-mode"):
            r(*args, torch.arange(2))
        with pytest.raises(ValueError, match="cuda"):  # a level alone is none
            r(q.detach(), k.detach(), torch.arange(2))


def test_attention_and_cache():
    c = paged.PagedCache(4, 16, 2, 64, device="cpu")
    i = lambda *s: torch.zeros(*s, dtype=torch.int32)
    q, k = torch.zeros(2, 3, 4, 64, dtype=torch.bfloat16), torch.zeros(3, 2, 64, dtype=torch.bfloat16)
    with forward_ad.dual_level():
        with pytest.raises(RuntimeError, match="tree_attention: no forward-mode"):
            speculative.tree_attention(_dual(q), c, i(2, 4), i(2))
        for args in ((_dual(k), k), (k, _dual(k))):
            with pytest.raises(RuntimeError, match="PagedCache.write: no forward-mode"):
                c.write(*args, torch.arange(3))
