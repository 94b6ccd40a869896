"""The 8-bit KV cache without a GPU: what its entry points refuse, and the restatement the GPU tests check against."""

from __future__ import annotations

import ctypes

import numpy as np
import pytest
import torch

from jitengine_amd import _lib, ops
from tests import kv8_ref as ref

X = ctypes.c_void_p(4096)  # (never dereferenced: every call here returns before a launch)
ODD = ctypes.c_void_p(4104)
EINVAL, EUNS, OK = _lib.JIT_EINVAL, _lib.JIT_EUNSUPPORTED, _lib.JIT_OK


def test_format_of_the_restatement():
    lut = ref.e4m3_values()
    torch8 = torch.arange(256, dtype=torch.uint8).view(torch.float8_e4m3fn).double()
    assert torch.equal(torch.nan_to_num(lut, nan=-1.0), torch.nan_to_num(torch8, nan=-1.0))
    x = torch.randn((64, 128), generator=torch.Generator().manual_seed(1), dtype=torch.float64).float()
    c, e = ref.quantise(x)
    back = lut[c] * torch.exp2(e.double())[:, None]
    # half an e4m3 step: 2^-4 of the value, or half the smallest step (2^-10) of the scale
    assert bool(((back - x).abs() <= torch.maximum(2.0 ** -4 * x.abs(), torch.exp2(e - 10.0)[:, None])).all())
    want = (x / torch.exp2(e.float())[:, None]).to(torch.float8_e4m3fn).view(torch.uint8)
    assert torch.equal(c, want.long())
    assert ref.scale_exp(torch.tensor([0.0, 448.0, 449.0, 224.0, 1e-300, 1.79e308], dtype=torch.float64)).tolist() == [
        0, 0, 1, -1, -100, 118]
    at = {ref.k_at(t, d) for t in range(16) for d in range(128)} | {ref.v_at(t, d) for t in range(16) for d in range(128)}
    assert at == set(range(4096))


def test_write_then_read_of_the_restatement():
    g = torch.Generator().manual_seed(2)
    pool = torch.zeros((3, 2, ops.KV8_RECORD), dtype=torch.uint8)
    k, v = (torch.randn((2, 2, 128), generator=g).to(torch.bfloat16) for _ in range(2))
    ref.write(pool, k, v, [37, 5])
    rk, rv = ref.read(pool, [0, 2])  # slot 5 is key 5 of page 0, slot 37 key 5 of page 2
    for x, r in ((k, rk), (v, rv)):
        x = x.double()
        assert bool(((r[:, 16 + 5] - x[0]).abs() <= 2.0 ** -4 * x[0].abs() + 2.0 ** -15).all())
        assert bool(((r[:, 5] - x[1]).abs() <= 2.0 ** -4 * x[1].abs() + 2.0 ** -15).all())


def _append(B=2, Hkv=4, pages=8, slots=X, pool=X):
    return _lib.lib().jit_kv8_append_paged(X, X, B, Hkv, slots, pool, pages, None)


def _fused(B=2, H=32, Hkv=4, pages=8, q=X):
    return _lib.lib().jit_qk_norm_rope_append_kv8(X, B, H, Hkv, X, X, 1e-6, X, X, X, X, pages, q, None)


def _decode(q=X, pool=X, pages=8, W=4, B=2, H=32, Hkv=4, max_len=64, ws=None, nb=0, out=X, lens=X):
    return _lib.lib().jit_paged_decode_attn_kv8(q, pool, pages, X, W, lens, B, H, Hkv, max_len, 0.1, ws, nb, out, None)


def _prefill(q=X, pool=X, pages=8, W=4, C=1, nblk=1, slots=0, max_len=4, units=1, H=32, Hkv=4, scale=0.1, ws=X, nb=1 << 40,
             out=X, unit=X, part=X, slot=X):
    return _lib.lib().jit_paged_prefill_attn_kv8(q, pool, pages, X, W, X, X, X, X, unit, part, slot, C, units, slots, X, X, X,
                                                 nblk, max_len, H, Hkv, scale, ws, nb, out, None)


def _tables(S=2, W=4, rows=2, free=None, n_free=-1, ctx=X, row_start=X, pos=X, status=X):
    return _lib.lib().jit_step_tables(ctx, X, S, X, W, rows, free, n_free, None, row_start, X, pos, X, X, status, None)


@pytest.mark.parametrize("call, want", [
    (lambda: _append(B=-1), EINVAL), (lambda: _append(Hkv=0), EINVAL), (lambda: _append(pages=0), EINVAL),
    (lambda: _append(slots=None), EINVAL), (lambda: _append(B=0, slots=None), OK), (lambda: _append(B=65536), EUNS),
    (lambda: _append(pool=ODD), EINVAL),
    (lambda: _fused(H=30), EINVAL), (lambda: _fused(Hkv=0), EINVAL), (lambda: _fused(B=-2), EINVAL),
    (lambda: _fused(q=None), EINVAL), (lambda: _fused(B=0, q=None), OK), (lambda: _fused(B=65536), EUNS),
    (lambda: _decode(B=-1), EINVAL), (lambda: _decode(H=30), EINVAL), (lambda: _decode(H=68, Hkv=4), EUNS),
    (lambda: _decode(max_len=-1), EINVAL), (lambda: _decode(W=0), EINVAL), (lambda: _decode(pages=0), EINVAL),
    (lambda: _decode(q=None), EINVAL), (lambda: _decode(lens=None), EINVAL), (lambda: _decode(B=0, q=None), OK),
    (lambda: _decode(W=4096, max_len=65536, ws=X, nb=16), EINVAL),  # a workspace too small for the chunks
    (lambda: _decode(q=ODD), EINVAL), (lambda: _decode(out=ODD), EINVAL), (lambda: _decode(pool=ODD), EINVAL),
    (lambda: _prefill(H=30), EINVAL), (lambda: _prefill(H=24, Hkv=8), EUNS), (lambda: _prefill(H=12, Hkv=4), EUNS),
    (lambda: _prefill(slots=-1), EINVAL), (lambda: _prefill(ws=None), EINVAL), (lambda: _prefill(nblk=1 << 30), EUNS),
    (lambda: _prefill(nb=32776 * 4 - 1), EINVAL), (lambda: _prefill(nb=32776 * 4, slots=8), EINVAL), (lambda: _prefill(units=0), EINVAL),
    (lambda: _prefill(part=None), EINVAL), (lambda: _prefill(slot=None), EINVAL), (lambda: _prefill(nblk=-1), EINVAL),
    (lambda: _prefill(scale=0.0), EINVAL), (lambda: _prefill(scale=-1.0), EINVAL), (lambda: _prefill(scale=float("nan")), EINVAL),
    (lambda: _prefill(unit=None), EINVAL), (lambda: _prefill(max_len=-1), EINVAL),
    (lambda: _prefill(C=0, q=None), OK), (lambda: _prefill(out=None), EINVAL), (lambda: _prefill(C=65536), EUNS),
    (lambda: _prefill(q=ODD), EINVAL), (lambda: _prefill(pool=ODD), EINVAL),
    (lambda: _tables(S=-1), EINVAL), (lambda: _tables(W=0), EINVAL), (lambda: _tables(rows=-1), EINVAL),
    (lambda: _tables(S=8193), EUNS), (lambda: _tables(ctx=None), EINVAL), (lambda: _tables(pos=None), EINVAL),
    (lambda: _tables(status=None), EINVAL), (lambda: _tables(n_free=3), EINVAL), (lambda: _tables(row_start=None), EINVAL),
    (lambda: _lib.lib().jit_kv8_copy_pages(X, 0, 4, X, X, 1, None), EINVAL),
    (lambda: _lib.lib().jit_kv8_copy_pages(None, 8, 4, X, X, 1, None), EINVAL),
    (lambda: _lib.lib().jit_kv8_copy_pages(None, 8, 4, None, None, 0, None), OK),
])
def test_contract_breaks_are_refused_before_any_launch(call, want):
    assert call() == want


def test_split_depends_on_the_length_alone():
    lib = _lib.lib()
    ck = {n: lib.jit_kv8_chunk_tokens(n) for n in (1, 512, 65536, 65537, 262144, 1 << 20, (1 << 31) - 1)}
    assert all(c % 128 == 0 and 128 <= c <= 4096 for c in ck.values())
    assert ck[1 << 20] == ck[(1 << 31) - 1] == 4096
    # the workspace holds the chunks of every length up to the bound
    for most in (1, 600, 65536, 70000, 300000, 1 << 20):
        have = lib.jit_kv8_decode_workspace_bytes(3, 32, most)
        for n in {1, most // 3 + 1, most - 1, most, min(most, 65536), min(most, 65537)}:
            chunks = -(-n // lib.jit_kv8_chunk_tokens(n)) if n > 0 else 0
            assert chunks <= 1 or have >= 3 * chunks * 32 * 130 * 4
    assert lib.jit_kv8_decode_workspace_bytes(3, 32, 0) == 0 and lib.jit_kv8_decode_workspace_bytes(-1, 32, 5) == -1


def test_the_ops_refuse_what_they_cannot_take():
    pool = ops.kv8_pool(4, 2, "cpu")
    assert pool.shape == (4, 2, ops.KV8_RECORD) and ops.is_kv8(pool) and not ops.is_kv8(torch.zeros(1, dtype=torch.bfloat16))
    with pytest.raises(ValueError):
        ops.kv8_pool(0, 2, "cpu")
    i = torch.zeros(2, dtype=torch.int32)
    kv = torch.zeros((2, 2, 128), dtype=torch.bfloat16)
    with pytest.raises(ValueError, match="device tensor"):
        ops.kv8_append_paged(pool, kv, kv, i)
    with pytest.raises(ValueError, match="device tensor"):
        ops.step_tables(i, i, torch.zeros((2, 4), dtype=torch.int32), 2)
    with pytest.raises(ValueError, match="device tensor"):
        ops.paged_decode_attention_kv8(kv, pool, torch.zeros((2, 4), dtype=torch.int32), i, 16, 0.1)


@pytest.mark.parametrize("seed", range(6))
def test_tables_of_the_restatement_never_share_a_slot(seed):
    import random

    r = random.Random(seed)
    S, W = r.randint(1, 9), r.randint(2, 12)
    ctx = [r.randint(0, 8 * W) for _ in range(S)]
    new = [r.choice([0, 1, 1, r.randint(0, 60)]) for _ in range(S)]
    perm = r.sample(range(1000), 1000)
    table = [[perm.pop() if j < -(-c // 16) else -1 for j in range(W)] for c in ctx]
    rows = sum(new) + r.choice([0, 3, -2 if sum(new) > 2 else 0])
    t = ref.step_tables(ctx, new, table, rows, free=perm[:r.randint(0, 12)])
    used = [s for s in t["slots"] if s >= 0]
    assert len(used) == len(set(used)) and t["row_start"][-1] == sum(new)
    assert sum(n - c for n, c in zip(t["lens"], ctx)) == len(used)


def _plan(ctx, length, H=32, Hkv=4):
    """(chunk_unit, chunk_part, chunk_slot, items in order) of jit_kv8_prefill_plan."""
    lib, C = _lib.lib(), len(ctx)
    a, b, tab = np.array(ctx, np.int32), np.array(length, np.int32), np.full((3, C + 1), -9, np.int32)
    args = a.ctypes.data, b.ctypes.data, C, H, Hkv, tab.ctypes.data
    n = lib.jit_kv8_prefill_plan(*args, None, 0)
    assert n >= 0
    blk = np.full((3, n), -9, np.int32)
    assert lib.jit_kv8_prefill_plan(*args, blk.ctypes.data, n) == n
    assert lib.jit_kv8_prefill_plan(*args, blk.ctypes.data, n + 1) == EINVAL
    return (*(t.tolist() for t in tab), list(zip(*blk.tolist())))


@pytest.mark.parametrize("H, Hkv", [(32, 4), (16, 16), (16, 1), (128, 16)])
@pytest.mark.parametrize("ctx, length", [
    ([0], [1]), ([8000], [16]), ([8192], [2048]), ([235, 0, 5834, 40000], [994, 3, 8, 700]), ([], []), ([262128], [16]),
])
def test_a_prompt_plan_covers_every_key_of_every_row_once(ctx, length, H, Hkv):
    first, part, slot, items = _plan(ctx, length, H, Hkv)
    bt = _lib.lib().jit_kv8_prefill_block_tokens(H, Hkv)
    assert bt == 128 * Hkv // H
    want, work = {}, []
    for c, (k, n) in enumerate(zip(ctx, length)):
        units = -(-(k + n) // 64)
        assert first[c + 1] - first[c] == units and 1 <= part[c] <= 192
        parts = -(-units // part[c])
        assert slot[c + 1] - slot[c] == (n * parts if parts > 1 else 0)
        for q0 in range(0, n, bt):
            nu = -(-(k + min(q0 + bt, n)) // 64)
            for p in range(-(-nu // part[c])):
                want[c, q0, p] = min(part[c], nu - p * part[c])
    assert first[0] == slot[0] == 0 and len(items) == len(want) and set(items) == set(want)
    work = [want[i] for i in items]
    assert work == sorted(work, reverse=True)


def test_a_chunk_is_cut_by_its_own_shape():
    alone = _plan([5834], [8])[1][0]
    assert _plan([235, 5834, 40000], [994, 8, 700])[1][1] == alone
    pu = _lib.lib().jit_kv8_prefill_part_units
    assert pu(0, 1, 32, 4) == 1 and pu(0, 500, 32, 4) == 8     # short sequences: one part
    assert pu(8000, 16, 32, 4) < 12                             # few rows, many keys: short parts
    assert pu(8192, 2048, 32, 4) == 160                         # enough rows: whole
    assert max(pu(c, 2048, 32, 4) for c in range(0, 262144, 4099)) <= 192
    assert pu(-1, 3, 32, 4) == -1 and pu(0, 0, 32, 4) == -1 and pu(0, 4, 30, 4) == -1


@pytest.mark.parametrize("ctx, length, H, want", [
    ([0], [0], 32, EINVAL), ([-1], [4], 32, EINVAL), ([0], [4], 12, EUNS), ([2 ** 31 - 1] * 80, [2 ** 31 - 1] * 80, 32, EUNS),
])
def test_a_prompt_plan_refuses_what_it_cannot_cut(ctx, length, H, want):
    a, b, tab = np.array(ctx, np.int32), np.array(length, np.int32), np.zeros((3, len(ctx) + 1), np.int32)
    assert _lib.lib().jit_kv8_prefill_plan(a.ctypes.data, b.ctypes.data, len(ctx), H, 4, tab.ctypes.data, None, 0) == want
    assert _lib.lib().jit_kv8_prefill_plan(None, b.ctypes.data, 1, 32, 4, tab.ctypes.data, None, 0) == EINVAL
