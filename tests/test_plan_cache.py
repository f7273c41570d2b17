"""The split plans kept between calls are bounded (a serving loop asks for another length every step)."""

from __future__ import annotations


def test_split_plans_kept_are_bounded(monkeypatch):
    from mxflashattn_b200 import _lib, backend

    monkeypatch.setattr(backend, "_LIB", [_lib.load()])
    monkeypatch.setattr(backend, "_PLANS", {})
    first = backend.kvcache_plan(1, 1, 8, 2, 128, 1)
    for n in range(1, 20001):
        backend.kvcache_plan(1, 1, 8, 2, 128, n)
    assert len(backend._PLANS) <= 4096
    assert backend.kvcache_plan(1, 1, 8, 2, 128, 1) == first
