"""check_status() of the 8-bit operators reports every call since the last check, on whatever stream it runs, and takes away
only what it reports."""

from __future__ import annotations

import pytest
import torch

from llm_inference_engine_b200 import _capi, cache8


class Word:
    """The device's word as the host sees it: reports of calls in flight land when the device is waited for."""

    def __init__(self, monkeypatch, in_flight):
        self.word, self.in_flight, self.waited = torch.zeros(1, dtype=torch.int32), in_flight, []
        monkeypatch.setattr(_capi, "_STATUS", {0: self.word})
        monkeypatch.setattr(torch.cuda, "synchronize", self.synchronize)

    def synchronize(self, device=None):
        self.waited.append(torch.device(device).index)
        self.word |= self.in_flight
        self.in_flight = 0


def test_calls_on_other_streams_are_waited_for(monkeypatch):
    w = Word(monkeypatch, 128)
    with pytest.raises(_capi.MuseError, match="page index outside"):
        cache8.check_status("cuda:0")
    assert w.waited == [0]
    cache8.check_status("cuda:0")   # reported once


def test_a_report_that_lands_behind_the_check_is_kept(monkeypatch):
    w = Word(monkeypatch, 256)
    real = torch.Tensor.item

    def item(self):   # another thread's call reports between the read and the clearing
        bits = real(self)
        if self is w.word and bits == 256:
            w.word |= 128
        return bits

    monkeypatch.setattr(torch.Tensor, "item", item)
    with pytest.raises(_capi.MuseError, match="lengths"):
        cache8.check_status("cuda:0")
    monkeypatch.setattr(torch.Tensor, "item", real)
    with pytest.raises(_capi.MuseError, match="page index outside"):
        cache8.check_status("cuda:0")
    cache8.check_status("cuda:0")


def test_a_new_word_is_zero_before_any_stream_gets_it(monkeypatch):
    order = []

    class Bind:
        set_status = staticmethod(lambda index, address: order.append("handed out"))

    zeros = torch.zeros

    def on_cpu(*size, device, dtype):
        order.append("made")
        return zeros(*size, dtype=dtype)

    monkeypatch.setattr(_capi, "_STATUS", {})
    monkeypatch.setattr(_capi, "_BIND", Bind)
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: False)
    monkeypatch.setattr(torch, "zeros", on_cpu)
    monkeypatch.setattr(torch.cuda, "synchronize", lambda device=None: order.append("waited"))
    address = _capi.status_ptr(0)
    assert order == ["made", "waited", "handed out"] and _capi.status_ptr(0) == address and len(order) == 3


@pytest.mark.gpu
def test_a_call_on_another_stream_is_reported():
    dev = torch.device("cuda:0")
    cache = cache8.new_cache(2, 1, 64, dev)
    q = torch.ones((1, 1, 64), device=dev, dtype=torch.bfloat16)
    table, lens = torch.tensor([[9]], dtype=torch.int32, device=dev), torch.tensor([5], dtype=torch.int32, device=dev)
    cache8.attention(q, cache, torch.zeros_like(table), lens)
    cache8.check_status(dev)
    side = torch.cuda.Stream(dev)
    with torch.cuda.stream(side):
        torch.cuda._sleep(200_000_000)   # about 0.1 s
        out = cache8.attention(q, cache, table, lens)
    with pytest.raises(_capi.MuseError, match="page index outside"):
        cache8.check_status(dev)
    assert bool((out == 0).all())
    cache8.check_status(dev)
