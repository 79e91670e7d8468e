"""Streams and lifetimes of the training operators, on stand-ins for streams and contexts; no GPU."""
import types

import pytest

torch = pytest.importorskip("torch")


class Kept:
    """what a call holds of a tensor: notes the streams that it is recorded on"""

    def __init__(self):
        self.on = []

    def record_stream(self, stream):
        self.on.append(stream)


def a_block(monkeypatch, made_on, now, gate=True):
    from unittest import mock

    from universal_differential_equations_amd import layers
    monkeypatch.setattr(layers, "Engine", mock.MagicMock())
    monkeypatch.setattr(layers, "current_raw_stream", lambda device: now)
    b = layers._Block.__new__(layers._Block)
    b.torch = types.SimpleNamespace(cuda=types.SimpleNamespace(current_stream=lambda device: "stream %d" % now))
    b.device, b.stream = torch.device("cuda", 0), made_on
    b.x, b.w, b.gate = Kept(), (Kept(), Kept(), Kept()), Kept() if gate else None
    return b


def test_everything_saved_is_kept_for_the_stream_of_its_pullback(monkeypatch):
    """x (which may be a copy that nobody but `saved` holds), weights, gate and up"""
    b = a_block(monkeypatch, made_on=7, now=9)
    b.bind()
    assert [t.on for t in (b.x, *b.w, b.gate)] == [["stream 9"]] * 5


def test_the_stream_they_were_made_on_needs_no_record(monkeypatch):
    for gate in (True, False):
        b = a_block(monkeypatch, made_on=7, now=7, gate=gate)
        b.bind()
        assert not any(t.on for t in (b.x, *b.w)) and (b.gate is None or not b.gate.on)
