"""Sizes past what the scoring and continuation operators' index arithmetic and launches cover: refused before anything runs."""

from __future__ import annotations

import ctypes

from jitengine_amd import _lib

D = ctypes.c_void_p(256)  # (never dereferenced)


def test_head_logprobs_refuses_rows_past_its_offsets():
    lib, U = _lib.lib(), _lib.JIT_EUNSUPPORTED
    for K in ((1 << 24) + 128, 1 << 28, (1 << 31) - 128):
        for V in (16, 32):
            assert lib.jit_head_logprobs(D, 1, K, D, V, D, D, D, D, D, 1 << 62, None) == U
            assert b"2^24" in lib.jit_last_error()
    assert lib.jit_head_logprobs(D, 128, 1 << 24, D, 16, D, D, D, D, D, 1 << 62, None) == U
    assert lib.jit_head_logprobs(D, 1, 1 << 24, D, 16, D, D, D, D, None, 0, None) == _lib.JIT_EINVAL  # (its workspace)
