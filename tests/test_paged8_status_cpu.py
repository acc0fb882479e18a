"""Status words of 8-bit caches (no GPU work)."""

import threading

import pytest
import torch

from multics_b200 import paged8
from multics_b200.paged8 import Paged8Cache


def _layers(n):
    c = Paged8Cache(2, 1, device="cpu")
    return [Paged8Cache.from_tensors(c.k, c.v, c.k_scale, c.v_scale) for _ in range(n)]


def test_every_cache_has_its_word():
    a, *rest = layers = _layers(600)
    assert len({c.status.data_ptr() for c in layers}) == 600
    a.status.fill_(4)
    for c in rest:
        c.check()
    with pytest.raises(ValueError, match="page pool"):
        a.check()
    a.check()


def test_caches_of_inference_mode_are_checked_outside():
    paged8._STATUS.clear()
    with torch.inference_mode():
        made = [*_layers(2), Paged8Cache(2, 1, device="cpu")]
    later, = _layers(1)
    for c in (*made, later):
        c.status.fill_(4)
        with pytest.raises(ValueError, match="page pool"):
            c.check()
        c.check()
        with torch.inference_mode():
            c.check()


def test_what_is_recorded_during_a_check_is_kept(monkeypatch):
    c, = _layers(1)
    late_record(c, monkeypatch)


def late_record(c, monkeypatch):
    """A kernel on another stream records a length while check() reads."""
    item, late = torch.Tensor.item, [2]

    def read(t):
        v = item(t)
        if late:
            c.status.bitwise_or_(late.pop())
        return v

    c.status.fill_(4)
    with monkeypatch.context() as m:
        m.setattr(torch.Tensor, "item", read)
        with pytest.raises(ValueError, match="page pool"):
            c.check()
    with pytest.raises(ValueError, match="block table"):
        c.check()
    c.check()


def test_a_given_word_is_shared():
    a = Paged8Cache(2, 1, device="cpu")
    b = Paged8Cache.from_tensors(a.k, a.v, a.k_scale, a.v_scale, a.status)
    assert b.status is a.status


def test_words_are_handed_out_once_to_threads():
    paged8._STATUS.clear()
    seen = []
    threads = [threading.Thread(target=lambda: seen.extend(_layers(300))) for _ in range(8)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert len({c.status.data_ptr() for c in seen}) == 2400
