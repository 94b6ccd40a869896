"""Scoring, searches and per-token log-probabilities of an engine: what is refused before anything runs (no GPU)."""

from __future__ import annotations

from types import SimpleNamespace

import pytest
import torch

from jitengine_amd import torch_ops
from jitengine_amd.engine import Engine
from jitengine_amd.kvpool import PoolExhausted
from jitengine_amd.model import MoEConfig


def _engine(pages=8, vocab=100, **kw):
    lm = SimpleNamespace(cfg=MoEConfig(layers=2), layers=[None, None], vocab=vocab, eos_ids=(3,))
    return Engine(lm, pages, prefill_chunk=32, max_step_tokens=32, device="cpu", allocate=False, **kw)


@pytest.mark.parametrize("n", [-1, 65])
def test_submit_refuses_alternatives_outside_the_range(n):
    eng = _engine()
    with pytest.raises(ValueError, match="logprobs"):
        eng.submit([1, 2], 4, logprobs=n)
    assert not eng.queue
    assert eng.submit([1, 2], 4, logprobs=64).top == 64 and eng.submit([1, 2], 4).top is None


def test_submit_refuses_more_alternatives_than_tokens():
    with pytest.raises(ValueError, match="logprobs"):
        _engine(vocab=10).submit([1, 2], 4, logprobs=11)


@pytest.mark.parametrize("args,match", [
    (([[1, 2]], 0, 4), "beams"), (([[1, 2]], 65, 4), "beams"), (([[1, 2]], 2, 0), "max_tokens"),
    (([[]], 2, 4), "empty"), (([[1, 100]], 2, 4), "token ids"), (([[-1]], 2, 4), "token ids"),
    (([[1]] * 5, 8, 4), "rows"),
])
def test_beam_search_refuses(args, match):
    eng = _engine()
    with pytest.raises(ValueError, match=match):
        eng.beam_search(*args)
    assert eng.pool.free_pages == 8 and not eng.pool.pages


def test_beam_search_of_no_prompts():
    assert _engine().beam_search([], 4, 4) == []


def test_searches_and_scores_past_the_pool_are_refused_and_hold_nothing():
    eng = _engine()
    with pytest.raises(PoolExhausted):
        eng.beam_search([[1] * 40], 4, 40)
    with pytest.raises(PoolExhausted):
        eng.score([1] * 200)
    eng.outstanding = 7  # (owed to admitted requests)
    with pytest.raises(PoolExhausted):
        eng.score([1] * 40)
    assert eng.pool.free_pages == 8 and not eng.pool.pages


def test_a_search_that_fails_gives_its_pages_back():
    eng = _engine(64)
    for call in (lambda: eng.beam_search([[1, 2]], 2, 4), lambda: eng.score([1, 2, 3])):
        with pytest.raises(AttributeError):  # (a model without weights)
            call()
        assert eng.pool.free_pages == 64 and not eng.pool.pages and not eng.pool.refs.any()


def test_score_of_a_single_token_and_of_none():
    assert _engine().score([5]) == []
    with pytest.raises(ValueError, match="empty"):
        _engine().score([])


def test_operators_are_registered_and_propagate_shapes():
    J, i32, f32, bf = torch.ops.jitengine, torch.int32, torch.float32, torch.bfloat16
    assert all(hasattr(J, n) for n in torch_ops.OPS_SCORING)

    def m(shape, dtype):
        return torch.empty(shape, dtype=dtype, device="meta")

    out = J.token_logprobs(m((3, 100), bf), m((3, 2), i32), 5)
    assert [(tuple(t.shape), t.dtype) for t in out] == [((3, 2), f32), ((3, 2), i32), ((3,), f32), ((3, 5), i32), ((3, 5), f32)]
    out = J.head_logprobs(m((7, 256), bf), m((1,), torch.uint8), 512, 256, m((7,), i32))
    assert out.shape == (3, 7) and out.dtype == f32
    out = J.beam_select(m((2, 3), f32), m((2, 3, 4), f32), m((2, 3, 4), i32), 5, None, None)
    assert [(tuple(t.shape), t.dtype) for t in out] == [((2, 5), i32), ((2, 5), i32), ((2, 5), f32), ((2, 5), i32)]
    out = J.pages_fork(m((2, 9), i32), m((2,), i32), m((6,), i32), m((50,), i32), m((20,), i32), m((1,), i32))
    assert [tuple(t.shape) for t in out] == [(6, 9), (6,), (6,), (6,), (4,)]
    assert J.kv_copy_pages_layers([m((4, 2, 2, 2048), bf)] * 2, m((1,), i32), m((1,), i32)) is None
