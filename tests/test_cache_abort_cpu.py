"""Leaving a step of a cache whose writing may have been replayed from a graph, without a GPU."""

import pytest
import torch

from rbf_attention_b200 import cache as cache_module
from rbf_attention_b200.cache import PagedCache


def _cache():
    return PagedCache(2, 2, 64, 3, 1000, device="cpu")


def _step(c, new):
    c.begin(new)
    c.end()


def _lengths(c):
    assert c.lengths.tolist() == [c.length(s) for s in range(3)]
    return c.lengths.tolist()


def test_a_step_is_taken_as_written_once_append_was_captured(monkeypatch):
    monkeypatch.setattr(cache_module.ops, "cache_append", lambda *a: None)
    c = _cache()
    rows = [torch.zeros(3, 2, 1, 64, dtype=torch.bfloat16)] * 2
    _step(c, [20, 30, 0])
    c.begin(1)
    c.append(0, *rows)                      # not captured
    c.end()
    c.begin([300, 1, 0])
    c.abort()                               # nothing written
    assert _lengths(c) == [21, 31, 1] and [len(h) for h in c._held] == [1, 1, 1]
    monkeypatch.setattr(cache_module.ops, "capturing", lambda device: True)
    c.begin(1)
    c.append(0, *rows)
    c.end()
    monkeypatch.setattr(cache_module.ops, "capturing", lambda device: False)
    c.begin([1, 0, 0])
    c.abort()                               # perhaps a replay
    assert _lengths(c) == [0, 32, 2] and c.free_pages == c.num_pages - 2


@pytest.mark.parametrize("appended", [False, True])
def test_the_caller_may_know(appended, monkeypatch):
    monkeypatch.setattr(cache_module.ops, "cache_append", lambda *a: None)
    c = _cache()
    _step(c, [20, 30, 5])
    for written, want in ((False, [20, 30, 5]), (True, [0, 0, 5])):
        c.begin([1, 300, 0])
        if appended:
            c.append(0, *[torch.zeros(3, 2, 300, 64, dtype=torch.bfloat16)] * 2)
        c.abort(written=written)
        assert _lengths(c) == want
        assert sorted(c._free) == [p for p, n in enumerate(c._users) if n == 0]
    assert c.free_pages == c.num_pages - 1
