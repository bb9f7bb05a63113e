"""Copies of a rotary embedding turn by their own frequencies: its descriptor
names the tensor that the copy holds."""

import copy
import pickle
import struct

import pytest
import torch

from voyager_amd import rotary


@pytest.mark.parametrize("way", [copy.deepcopy, lambda r: pickle.loads(pickle.dumps(r)), copy.copy])
def test_a_copy_names_its_own_frequencies(way, monkeypatch):
    seen = []

    class Entry:
        @staticmethod
        def vh_rope(descriptor, stream):
            seen.append(descriptor)
            return 0

    monkeypatch.setattr(rotary, "load", lambda: Entry)
    monkeypatch.setattr(rotary, "stream_on", lambda device: 0)
    first = rotary.Rotary(16, interleaved=True, scaling={"kind": "linear", "factor": 2.0}, device="cpu")
    second = way(first)
    x, positions = torch.zeros(1, 2, 3, 16), torch.arange(2)
    for r in (first, second):
        r(x, None, positions)
        address, = struct.unpack_from("@Q", seen[-1], len(seen[-1]) - 8)
        assert address == r.turns.data_ptr()
    rest = rotary._ROPE_REST.size
    assert seen[0][-rest:-8] == seen[1][-rest:-8] and torch.equal(first.turns, second.turns)


def test_frequencies_put_elsewhere_are_followed(monkeypatch):
    seen = []
    monkeypatch.setattr(rotary, "load", lambda: type("Entry", (), {"vh_rope": staticmethod(lambda d, s: seen.append(d) or 0)}))
    monkeypatch.setattr(rotary, "stream_on", lambda device: 0)
    r = rotary.Rotary(8, device="cpu")
    r.turns = r.turns.clone()
    r(torch.zeros(1, 2, 3, 8), None, torch.arange(2))
    assert struct.unpack_from("@Q", seen[0], len(seen[0]) - 8)[0] == r.turns.data_ptr()


def test_frequencies_on_another_device_are_refused(monkeypatch):
    monkeypatch.setattr(rotary, "load", lambda: type("Entry", (), {"vh_rope": staticmethod(lambda d, s: 0)}))
    monkeypatch.setattr(rotary, "stream_on", lambda device: 0)
    r = rotary.Rotary(8, device="cpu")
    args = torch.zeros(1, 2, 3, 8), None, torch.arange(2)
    r(*args)
    r.turns = r.turns.to("meta")
    with pytest.raises(ValueError, match="frequencies on meta"):
        r(*args)
