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


def test_launches_past_2_32_threads_are_refused():
    lib, U = _lib.lib(), _lib.JIT_EUNSUPPORTED
    for B in (1 << 24, (1 << 31) - 1):
        assert lib.jit_token_logprobs(D, 0, B, 8, 8, D, 1, 2, D, D, D, D, D, None, 0, None) == U
        assert b"2^24 - 1 rows" in lib.jit_last_error()
    for G in (1 << 26, (1 << 31) - 1):
        assert lib.jit_beam_select(D, D, D, None, None, 0, G, 1, 4, 1, D, D, D, D, None) == U
    for S, N, W in ((8192, 1, 1 << 19), (0, 8192, 1 << 26)):
        assert lib.jit_pages_fork(D, D, S, W, D, N, D, 16, D, 16, D, D, D, D, D, D, D, 1 << 62, None) == U
