"""Sizes past what the scoring and continuation operators' index arithmetic and launches cover: refused before anything runs."""

from __future__ import annotations

import ctypes
from types import SimpleNamespace

import pytest
import torch

from jitengine_amd import _lib, ops

D = ctypes.c_void_p(256)  # (never dereferenced)


def test_head_logprobs_refuses_rows_past_its_offsets():
    lib, U = _lib.lib(), _lib.JIT_EUNSUPPORTED
    for K in ((1 << 24) + 128, 1 << 28, (1 << 31) - 128):
        for V in (16, 32):
            assert lib.jit_head_logprobs(D, 1, K, D, V, D, D, D, D, D, 1 << 62, None) == U
            assert b"2^24" in lib.jit_last_error()
    assert lib.jit_head_logprobs(D, 128, 1 << 24, D, 16, D, D, D, D, D, 1 << 62, None) == U
    assert lib.jit_head_logprobs(D, 1, 1 << 24, D, 16, D, D, D, D, None, 0, None) == _lib.JIT_EINVAL  # (its workspace)


def test_launches_past_2_32_threads_are_refused():
    lib, U = _lib.lib(), _lib.JIT_EUNSUPPORTED
    for B in (1 << 24, (1 << 31) - 1):
        assert lib.jit_token_logprobs(D, 0, B, 8, 8, D, 1, 2, D, D, D, D, D, None, 0, None) == U
        assert b"2^24 - 1 rows" in lib.jit_last_error()
    for G in (1 << 26, (1 << 31) - 1):
        assert lib.jit_beam_select(D, D, D, None, None, 0, G, 1, 4, 1, D, D, D, D, None) == U
    for S, N, W in ((8192, 1, 1 << 19), (0, 8192, 1 << 26)):
        assert lib.jit_pages_fork(D, D, S, W, D, N, D, 16, D, 16, D, D, D, D, D, D, D, 1 << 62, None) == U


BIG = 2 ** 32 + 8  # (cut to 32 bits: 8)


def _meta(*shape, dtype=torch.int32):
    return torch.empty(shape, dtype=dtype, device="meta")


@pytest.fixture
def on_device(monkeypatch):
    """Tensors without memory pass for device tensors, and nothing is launched."""
    def launched(*a):
        raise AssertionError("launched")

    monkeypatch.setattr(ops, "_take", lambda *t: 0)
    monkeypatch.setattr(ops, "_launch", launched)


@pytest.mark.parametrize("call", [
    lambda: ops.token_logprobs(_meta(1, BIG, dtype=torch.bfloat16)),
    lambda: ops.token_logprobs(_meta(BIG, 8, dtype=torch.bfloat16), _meta(BIG)),
    lambda: ops.token_logprobs(_meta(1, 8, dtype=torch.bfloat16), top=BIG),
    lambda: ops.token_logprobs(_meta(1, 8, dtype=torch.bfloat16), top=-BIG),
    lambda: ops.beam_select(_meta(BIG, 1, dtype=torch.float32), _meta(BIG, 1, 1, dtype=torch.float32), _meta(BIG, 1, 1)),
    lambda: ops.beam_select(_meta(1, 1, dtype=torch.float32), _meta(1, 1, BIG, dtype=torch.float32), _meta(1, 1, BIG)),
    lambda: ops.beam_select(_meta(1, 1, dtype=torch.float32), _meta(1, 1, 1, dtype=torch.float32), _meta(1, 1, 1), width=BIG),
    lambda: ops.beam_select(_meta(1, 1, dtype=torch.float32), _meta(1, 1, 1, dtype=torch.float32), _meta(1, 1, 1), eos=_meta(BIG)),
    lambda: ops.pages_fork(_meta(1, 4), _meta(1), _meta(BIG), _meta(16), _meta(16), _meta(1)),
    lambda: ops.pages_fork(_meta(1, 4), _meta(1), _meta(2), _meta(BIG), _meta(16), _meta(1)),
    lambda: ops.pages_fork(_meta(1, 4), _meta(1), _meta(2), _meta(16), _meta(BIG), _meta(1)),
    lambda: ops.kv_copy_pages_layers(SimpleNamespace(device=0), _meta(BIG), _meta(BIG)),
    lambda: ops.token_logprobs_workspace_bytes(1, BIG), lambda: ops.head_logprobs_workspace_bytes(BIG, 128, 16),
])
def test_sizes_past_32_bits_are_refused_not_cut(call, on_device):
    with pytest.raises(_lib.UnsupportedShape, match=r"2\^31"):
        call()
