"""What the kernels' sources have to say to the compiler, read without a GPU."""

import glob
import os
import re

import pytest

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "voyager-compiler-2_amd", "csrc")


def statements():
    for path in sorted(glob.glob(os.path.join(CSRC, "*"))):
        for m in re.finditer(r"\basm\b(?:\s+volatile)?\s*\((.*?)\)\s*;", open(path).read(), re.S):
            yield os.path.basename(path), m.group(1)


def test_statements_are_found():
    assert any("offen lds" in text for _, text in statements())


@pytest.mark.parametrize("path,text", [s for s in statements() if "offen lds" in s[1] or re.search(r"\bm0\b", s[1])])
def test_assembly_declares_m0(path, text):
    """Loads to LDS read M0, which the compiler uses as well: it is an operand, not written behind its back."""
    assert '"{m0}"' in text and not re.search(r"s_mov\w*\s+m0", text), f"{path}: {text}"
