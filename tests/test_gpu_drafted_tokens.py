"""The drafted-token operators together, as examples/drafted_tokens.py runs
them: with the target's best tokens, a drafted text is one that the model, in
one pass over the whole of it, finds best token by token."""

import os
import sys

import pytest
import torch

sys.path.insert(0, os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "examples"))

pytestmark = pytest.mark.gpu


def _texts(told, count):
    return [[x for s in range(told.shape[0]) for x in told[s, i, : int(count[s, i])].tolist()] for i in range(told.shape[1])]


# The model's activations and its last product are bfloat16, rounded about a
# dozen times on the way (the last time at values up to 8), in an order that
# goes by the batch's shape: a choice between tokens closer than this is open.
OPEN = 12**0.5 * 8 * 2.0**-8


@pytest.mark.parametrize("fmt", ["fp8_e4m3", "int8", None])
@pytest.mark.parametrize("depth", [0, 3])
def test_each_token_is_the_models_best(fmt, depth):
    import drafted_tokens as ex

    model = ex.Model(fmt=fmt)
    prompt = torch.randint(0, 512, (3, 21), generator=torch.Generator().manual_seed(5)).cuda()
    told, count = ex.generate(model, prompt, steps=10, depth=depth, temperature=0)
    if depth:
        assert max(map(len, _texts(told, count))) > 10  # drafts were kept
    for i, text in enumerate(_texts(told, count)):
        whole = torch.tensor([prompt[i].tolist() + text]).cuda()
        n = whole.shape[1]
        with torch.no_grad():
            logits = model(whole, torch.arange(n).cuda(), model.caches(8, 16), torch.arange(8).int().cuda()[None],
                           torch.zeros(1, dtype=torch.int32).cuda())[0, prompt.shape[1] - 1: -1]
        short = logits.max(-1).values - logits.gather(1, torch.tensor(text).cuda()[:, None])[:, 0]
        assert float(short.max()) <= OPEN, f"sequence {i}: {short.tolist()}"


def test_sampled_tokens_end_inside_the_vocabulary():
    import drafted_tokens as ex

    told, count = ex.generate(ex.Model(), torch.zeros(2, 1, dtype=torch.int64, device="cuda"), steps=6, branch=3, depth=2)
    assert bool((count >= 1).all()) and bool((count <= 3).all())
    for text in _texts(told, count):
        assert all(0 <= x < 512 for x in text)


def test_balanced_trees():
    import drafted_tokens as ex

    assert ex.balanced(2, 2) == ([-1, 0, 0, 1, 1, 2, 2], [0, 1, 1, 2, 2, 2, 2])
    assert ex.balanced(0, 5) == ([-1], [0])
