"""The 8-bit cache in the pool, the model and the engine: bookkeeping, refusals and registration (CPU)."""

from __future__ import annotations

import ctypes
from types import SimpleNamespace

import numpy as np
import pytest
import torch

from jitengine_amd import _lib, ops, torch_ops
from jitengine_amd import model as M
from jitengine_amd.engine import Engine
from jitengine_amd.kvpool import KVPool

CFG = M.MoEConfig(layers=1, experts=32)


def test_pool_holds_records_and_charges_their_bytes():
    p, b = KVPool(2, 6, 4, "cpu", kv8=True), KVPool(2, 6, 4, "cpu")
    assert [tuple(t.shape) for t in p.pools] == [(6, 4, ops.KV8_RECORD)] * 2
    assert all(ops.is_kv8(t) for t in p.pools) and not any(ops.is_kv8(t) for t in b.pools)
    assert p.page_bytes == p.pools[0][0].nbytes == 4 * 4224 and b.page_bytes == b.pools[0][0].nbytes
    lm = SimpleNamespace(cfg=SimpleNamespace(kv_heads=4, heads=32), layers=[None, None], vocab=100, eos_ids=(99,),
                         final_norm=torch.zeros(1))
    e = Engine(lm, 8, prefill_chunk=8, allocate=False, kv8=True)
    assert e.pool.kv8 and not Engine(lm, 8, prefill_chunk=8, allocate=False).pool.kv8
    with pytest.raises(ValueError, match="8192"):
        Engine(lm, 8, prefill_chunk=8, max_step_tokens=8193, allocate=False, kv8=True)
    Engine(lm, 8, prefill_chunk=8, max_step_tokens=8193, allocate=False)


def test_a_state_of_the_other_kind_is_refused():
    pool8, pool16 = ops.kv8_pool(2, 4, "cpu"), KVPool(1, 2, 4, "cpu").pools[0]
    with pytest.raises(ValueError, match="8-bit"):
        M._over_kv8(pool8, SimpleNamespace(kv8=None))
    with pytest.raises(ValueError, match="bf16"):
        M._over_kv8(pool16, SimpleNamespace(kv8=object()))
    assert M._over_kv8(pool8, SimpleNamespace(kv8=object())) and not M._over_kv8(pool16, SimpleNamespace(kv8=None))


@pytest.mark.parametrize("pos", [[31, 32], [-1, 3]])
def test_positions_outside_the_page_table_are_refused(pos):
    with pytest.raises(ValueError, match="outside"):
        M.make_step_state(CFG, pos, torch.zeros((2, 2), dtype=torch.int32), kv8=True)


@pytest.mark.parametrize("chunks, dec, dec_width, match", [
    ([(1, 0, 4)], [], 2, "do not match"),    # a chunk of a sequence that the table does not have
    ([(-1, 0, 4)], [], 2, "do not match"),
    ([(0, 0, 4)], [3], 4, "width"),          # two tables of unequal width
    ([(0, 20, 13)], [], 2, "outside"),       # 33 positions in 2 pages
    ([(0, 0, 4)], [32], 2, "outside"),
])
def test_mixed_steps_that_do_not_fit_their_tables_are_refused(chunks, dec, dec_width, match):
    with pytest.raises(ValueError, match=match):
        M.make_mixed_state(CFG, chunks, np.zeros((1, 2), np.int32), dec, np.zeros((len(dec), dec_width), np.int32),
                           "cpu", kv8=True)


def test_native_layer_calls_refuse_what_they_cannot_run():
    lib = _lib.lib()
    lay = _lib.Layer(2048, 32, 4, 32, 8, 768, 1, 1e-6, 0.1)
    for name, _ in lay._fields_[9:]:
        setattr(lay, name, 256)  # (never dereferenced)
    one = ctypes.c_void_p(256)

    def decode(step, x=one, defer=0, y=one):
        return lib.jit_decode_layer_kv8(lay, step, one, 1, x, None, None, None, defer, None, one, y, None, None)

    def mixed(step, x=one):
        return lib.jit_mixed_layer_kv8(lay, step, one, 1, x, one, one, None)

    assert decode(None) == _lib.JIT_EINVAL and mixed(None) == _lib.JIT_EINVAL
    assert decode(_lib.Kv8Step(prompt_rows=1, B=1)) == _lib.JIT_EINVAL and b"prompt" in lib.jit_last_error()
    assert decode(_lib.Kv8Step(B=0)) == _lib.JIT_EINVAL
    assert decode(_lib.Kv8Step(B=2), defer=1) == _lib.JIT_EINVAL and b"one row" in lib.jit_last_error()
    assert decode(_lib.Kv8Step(B=1), x=None) == _lib.JIT_EINVAL and b"null" in lib.jit_last_error()
    assert mixed(_lib.Kv8Step(prompt_rows=-1, B=3)) == _lib.JIT_EINVAL
    assert mixed(_lib.Kv8Step(B=1), x=None) == _lib.JIT_EINVAL


def test_operators_are_registered_and_propagate_shapes():
    J, i32, bf = torch.ops.jitengine, torch.int32, torch.bfloat16
    assert all(hasattr(J, n) for n in torch_ops.OPS_KV8)

    def m(shape, dtype):
        return torch.empty(shape, dtype=dtype, device="meta")

    pool, table = m((64, 4, ops.KV8_RECORD), torch.uint8), m((3, 8), i32)
    t = J.step_tables(m((3,), i32), m((3,), i32), table, 20, m((5,), i32), None)
    assert [tuple(x.shape) for x in t] == [(4,), (20,), (20,), (20,), (3,), (4,)]
    q = J.qk_norm_rope_append_kv8(m((20, 40 * 128), bf), 32, 4, m((128,), bf), m((128,), bf), 1e-6,
                                  m((64,), torch.float32), t[2], t[3], pool)
    assert q.shape == (20, 32, 128) and q.dtype == bf
    assert J.paged_decode_attention_kv8(q[:3], pool, table, t[4], 99, 0.1, m((64,), torch.uint8)).shape == (3, 32, 128)
    out = J.paged_prefill_attention_kv8(q, pool, table, m((4, 1), i32), m((3, 2), i32), m((3, 2), i32), [0, 0, 20], 1, 0,
                                        0.1, m((64,), torch.uint8))
    assert out.shape == q.shape and out.dtype == bf
    assert J.kv8_append_paged(pool, m((20, 4, 128), bf), m((20, 4, 128), bf), t[3]) is None
    assert J.kv8_copy_pages(pool, m((2,), i32), m((2,), i32)) is None
