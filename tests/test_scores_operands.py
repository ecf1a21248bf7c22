"""How a call of the operators on rows of scores orders the streams of its operands, without a GPU: the streams are stand-ins
that note who waits for whom."""

import contextlib
from types import SimpleNamespace

import pytest

from octex_amd import _arrays, _lib
from octex_amd import scores as S


class Stream:
    def __init__(self, name, notes):
        self.name, self.notes = name, notes

    def wait_stream(self, other):
        self.notes.append(f"{self.name} waits for {other.name}")


class Tensor:
    is_cuda = True


@pytest.fixture()
def call(monkeypatch):
    """A call on the stream `side` (7) of a framework, where torch's current stream is another (5)."""
    notes = []
    streams = {h: Stream(n, notes) for h, n in ((0, "null"), (5, "current"), (7, "side"), (9, "third"))}
    c = S._Call.__new__(S._Call)
    c.torch = SimpleNamespace(Tensor=Tensor, from_dlpack=lambda a: Tensor(), as_tensor=lambda a, device: Tensor(),
                              cuda=SimpleNamespace(current_stream=lambda device: streams[5], default_stream=lambda d: streams[0],
                                                   ExternalStream=lambda h, device: streams[h],
                                                   stream=lambda s: contextlib.nullcontext()))
    c.device, c.stream, c.side, c.others = None, 7, streams[7], ()
    monkeypatch.setattr(S, "_entry", lambda name: lambda *args: notes.append("launch") or _lib.CUVS_SUCCESS)
    return c, notes, streams


class Interface:
    def __init__(self, stream):
        self.__cuda_array_interface__ = dict(shape=(2, 2), typestr="<f4", data=(0, False), version=3, stream=stream)


def test_torch_operands_of_another_frameworks_call(call):
    c, notes, _ = call
    c.array(Tensor()), c.array(Tensor())
    c.run("any")
    assert notes == ["side waits for current", "launch", "current waits for side"]


def test_interfaces_name_their_streams(call):
    c, notes, streams = call
    c.array(Interface(9)), c.array(Interface(7)), c.array(Interface(None)), c.array(Interface(1))
    c.run("any")
    assert notes == ["side waits for third", "side waits for null", "launch", "third waits for side", "null waits for side"]


def test_torch_operands_of_a_torch_call(call):
    c, notes, _ = call
    c.stream, c.side = 5, None
    c.array(Tensor())
    c.run("any")
    assert notes == ["launch"]  # nothing is added to the ordinary call
    c.array(Interface(9))
    c.run("any")
    assert notes[1:] == ["current waits for third", "launch", "third waits for current"]


class Older:
    """An interface of a version that had no stream yet."""

    __cuda_array_interface__ = dict(shape=(2, 2), typestr="<f4", data=(0, False), version=2)


class OlderWithExport(Older):
    def __dlpack__(self, **kw):
        raise NotImplementedError


def test_interfaces_without_a_stream_are_ordered_on_the_null_stream(call):
    assert _arrays.named_stream(Older()) == 0 and _arrays.named_stream(OlderWithExport()) is None
    c, notes, _ = call
    c.array(Older()), c.array(OlderWithExport())
    c.run("any")
    assert notes == ["side waits for null", "launch", "null waits for side"]


def test_named_streams():
    assert _arrays.named_stream(Interface(1)) == 0 and _arrays.named_stream(Interface(9)) == 9
    assert _arrays.named_stream(Interface(None)) is None and _arrays.named_stream(object()) is None
