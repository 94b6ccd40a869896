"""Refusals and host contracts of the scoring and continuation operators: every call here returns before a launch."""

from __future__ import annotations

import ctypes

import numpy as np
import pytest
import torch

from jitengine_amd import _lib, ops
from tests.scoring_ref import beams_ref, fork_ref, rows_ref

D = ctypes.c_void_p(256)  # (never dereferenced)


def test_token_logprobs_contract():
    lib = _lib.lib()

    def call(B=1, V=100, stride=100, tokens=D, m=1, top=5, x=D, ws=D, nb=1 << 20, lp=D, ids=D):
        return lib.jit_token_logprobs(x, 0, B, V, stride, tokens, m, top, lp, D, D, ids, D, ws, nb, None)

    E, U = _lib.JIT_EINVAL, _lib.JIT_EUNSUPPORTED
    assert call(B=-1) == call(V=0) == call(m=-1) == call(top=-1) == call(stride=99) == E
    assert call(top=101) == E and b"top=101" in lib.jit_last_error()
    assert call(top=65) == call(m=65) == U
    assert call(V=(1 << 30) + 1, stride=1 << 31) == U
    assert call(tokens=None) == call(x=None) == call(lp=None) == call(ids=None) == E
    assert call(x=ctypes.c_void_p(257)) == E
    need = lib.jit_token_logprobs_workspace_bytes(1, 100000, 1, 5)
    assert need > 0 and lib.jit_token_logprobs_workspace_bytes(2048, 100000, 1, 5) == 0
    assert lib.jit_token_logprobs_workspace_bytes(1, 0, 1, 5) == -1
    assert call(V=100000, stride=100000, nb=need - 1) == call(V=100000, stride=100000, ws=None) == E
    assert call(V=100000, stride=100000, ws=ctypes.c_void_p(264)) == E
    assert call(B=0) == _lib.JIT_OK


def test_head_logprobs_contract():
    lib = _lib.lib()

    def call(T=3, K=128, V=32, x=D, ws=D, nb=1 << 40, lp=D):
        return lib.jit_head_logprobs(x, T, K, D, V, D, lp, D, D, ws, nb, None)

    E, U = _lib.JIT_EINVAL, _lib.JIT_EUNSUPPORTED
    assert call(T=-1) == call(K=0) == call(V=0) == E
    assert call(K=192) == call(V=40) == call(T=(1 << 20) + 1) == U
    assert call(x=None) == call(lp=None) == call(x=ctypes.c_void_p(264)) == call(ws=None) == call(nb=16) == E
    assert call(T=0) == _lib.JIT_OK
    assert lib.jit_head_logprobs_workspace_bytes(-1, 128, 32) == -1


def test_beam_select_contract():
    lib = _lib.lib()

    def call(G=1, n=2, m=3, w=2, e=0, eos=None, s=D):
        return lib.jit_beam_select(s, D, D, None, eos, e, G, n, m, w, D, D, D, D, None)

    E, U = _lib.JIT_EINVAL, _lib.JIT_EUNSUPPORTED
    assert call(G=-1) == call(n=0) == call(m=0) == call(w=0) == call(e=-1) == call(e=1) == call(s=None) == E
    assert call(w=65) == call(n=64, m=65) == U
    assert call(G=0) == _lib.JIT_OK


def test_pages_fork_contract():
    lib = _lib.lib()

    def call(S=2, W=4, N=2, P=16, F=16, table=D, refs=D, ws=D, nb=1 << 20):
        return lib.jit_pages_fork(table, D, S, W, D, N, refs, P, D, F, D, D, D, D, D, D, ws, nb, None)

    E, U = _lib.JIT_EINVAL, _lib.JIT_EUNSUPPORTED
    assert call(S=-1) == call(N=-1) == call(W=0) == call(P=0) == call(F=-1) == E
    assert call(S=8193) == call(N=8193) == call(W=(1 << 26) + 1) == call(P=(1 << 27) + 1) == U
    assert call(table=None) == call(refs=None) == call(ws=None) == call(nb=8) == call(ws=ctypes.c_void_p(264)) == E
    assert lib.jit_pages_fork_workspace_bytes(2, 2, 0) == -1


def test_copy_layers_contract():
    lib = _lib.lib()
    pools = (ctypes.c_void_p * 2)(256, 512)

    def call(p=pools, L=2, P=4, b=32768, src=D, n=1):
        return lib.jit_kv_copy_pages_layers(p, L, P, b, src, D, n, None)

    E = _lib.JIT_EINVAL
    assert call(L=-1) == call(P=0) == call(b=0) == call(n=-1) == call(p=None) == call(src=None) == E
    assert call(b=40) == _lib.JIT_EUNSUPPORTED
    assert call(p=(ctypes.c_void_p * 2)(256, 520)) == call(p=(ctypes.c_void_p * 2)(256, None)) == E
    assert b"layer 1" in lib.jit_last_error()
    assert call(n=0) == call(L=0) == _lib.JIT_OK


def test_host_functions_refuse_before_a_launch():
    x, t = torch.zeros((2, 8)), torch.zeros(2, dtype=torch.int32)
    with pytest.raises(ValueError, match="bf16 or fp32"):
        ops.token_logprobs(x.double(), t)
    with pytest.raises(ValueError, match="adjacent"):
        ops.token_logprobs(x.t(), t)
    with pytest.raises(ValueError, match="adjacent"):
        ops.token_logprobs(x[0], t)
    with pytest.raises(ValueError, match="device tensor"):
        ops.token_logprobs(x, t)
    with pytest.raises(_lib.UnsupportedShape):
        ops.head_logprobs(x.bfloat16(), object(), t)
    with pytest.raises(ValueError, match="device tensor"):
        ops.beam_select(x, torch.zeros((2, 8, 1)), torch.zeros((2, 8, 1), dtype=torch.int32))
    with pytest.raises(ValueError, match="must be torch.int32"):
        ops.pages_fork(x, t, t, t, t, t)
    with pytest.raises(ValueError, match="at least one"):
        ops.pool_layers([])
    with pytest.raises(ValueError, match="KV pool"):
        ops.pool_layers([torch.zeros((2, 1, 2, 5), dtype=torch.bfloat16)])


def test_the_references_agree_with_torch_and_with_counts():
    """The plain forms that the kernels are tested against, on cases that can be said by hand."""
    x = torch.tensor([[0.0, 1.0, 1.0, -np.inf], [2.0, 2.0, 2.0, 2.0], [-np.inf] * 4])
    lp, rank, ent, ids, tlp = rows_ref(x, torch.tensor([[2, 3], [1, 9], [0, 3]]), 3)
    want = torch.log_softmax(x[:2].double(), -1)
    assert torch.allclose(lp[0, 0], want[0, 2]) and lp[0, 1] == -np.inf and lp[1, 1] == 0
    assert rank.tolist() == [[1, 3], [1, -1], [0, 3]] and ids.tolist() == [[1, 2, 0], [0, 1, 2], [0, 1, 2]]
    assert torch.allclose(ent[1], torch.log(torch.tensor(4.0).double())) and ent[2] == 0
    p, t, s, d = beams_ref(np.float32([[-1, -2]]), np.float32([[[-1, -3], [0, -1]]]), np.int32([[[5, 6], [7, -1]]]), 4,
                           np.int32([[0, 0]]), (7,))
    assert p.tolist() == [[0, 1, 0, -1]] and t.tolist() == [[5, 7, 6, -1]] and d.tolist() == [[0, 1, 0, 1]]
    # two sequences of 20 tokens that share page 3: both go on from the first, which keeps its last page once
    new, nl, src, dst, status, refs, free = fork_ref([[3, 1], [3, 2]], [20, 20], [0, 0], [0, 1, 1, 2], [3, 1, 2, 0], 3)
    assert new.tolist() == [[3, 1], [3, 0]] and src == [-1, 1] and dst == [-1, 0] and refs == [1, 1, 0, 2]
    assert status == [1, 3, 0, 0] and free[3:] == [2]
