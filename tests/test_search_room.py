"""What scores and searches do to stored prefixes when there is no room for them (no GPU)."""

from __future__ import annotations

from types import SimpleNamespace

import pytest

from jitengine_amd.engine import Engine
from jitengine_amd.kvpool import PoolExhausted
from jitengine_amd.model import MoEConfig


def _engine(pages):
    lm = SimpleNamespace(cfg=MoEConfig(layers=2), layers=[None, None], vocab=100, eos_ids=(3,))
    return Engine(lm, pages, prefill_chunk=32, max_step_tokens=32, device="cpu", allocate=False)


def _store(eng, n, sid):
    """A stored prefix of n tokens, its sequence gone on holding the pages if `sid` is kept."""
    eng.pool.reserve(sid, n)
    eng.store.insert([len(eng.store.entries)] * n, eng.pool.pages[sid])


def test_what_cannot_fit_evicts_nothing():
    eng = _engine(16)
    for sid in ("a", "b"):
        _store(eng, 64, sid)
        eng.pool.release(sid)
    assert eng.store.held_alone() == 8 and eng.pool.free_pages == 8
    for call in (lambda: eng.score([1] * 300), lambda: eng.beam_search([[1] * 100], 4, 200)):
        with pytest.raises(PoolExhausted):
            call()
        assert len(eng.store.entries) == 2 and eng.pool.free_pages == 8
    eng.outstanding = 10  # (owed to admitted requests)
    with pytest.raises(PoolExhausted, match="6 free or held"):
        eng.score([1] * 120)
    assert len(eng.store.entries) == 2


def test_pages_that_a_sequence_holds_too_do_not_count():
    eng = _engine(16)
    _store(eng, 64, "a")
    _store(eng, 80, "b")
    eng.store.insert([9] * 32, eng.pool.pages["b"])  # (a second entry over b's first pages)
    eng.pool.release("b")
    assert eng.store.held_alone() == 5 and eng.pool.free_pages == 7
    with pytest.raises(PoolExhausted):
        eng.score([1] * (13 * 16))
    assert len(eng.store.entries) == 3
    with pytest.raises(AttributeError):  # (a model without weights: there was room for it)
        eng.score([1] * (12 * 16))
    assert eng.pool.free_pages == 12 and not eng.store.entries
