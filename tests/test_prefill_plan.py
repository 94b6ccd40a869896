"""Plans of prompt attention on the host: the work items of a bf16 pool restated as a loop, and which kinds of pool a
plan serves."""

from __future__ import annotations

import numpy as np
import pytest
import torch

from jitengine_amd import _lib, ops

EINVAL, EUNSUPPORTED = -1, -2


def _items(chunks, H, Hkv):
    """(chunk, first token, part) of every row block and key part, the most 128-key steps first."""
    lib = _lib.lib()
    bt, part = lib.jit_prefill_block_tokens(H, Hkv), lib.jit_prefill_part_keys() // 128
    items = []
    for c, (_, ctx, n) in enumerate(chunks):
        for q0 in range(0, n, bt):
            keys = ctx + min(q0 + bt, n)
            steps = -(-keys // 128)
            for p in range(-(-steps // part)):
                items.append((min(steps, (p + 1) * part) - p * part, keys, c, q0, p))
    items.sort(key=lambda it: (-it[0], -it[1]))  # (stable)
    return [it[2:] for it in items]


CHUNKS = [
    [], [(0, 0, 1)], [(3, 0, 512)], [(0, 8192, 2048)], [(0, 262000, 144)], [(0, 6143, 1), (1, 6144, 1), (2, 6112, 33)],
    [(i, 577 * i, 300 + 41 * i) for i in range(9)], [(0, 0, 64)] * 5 + [(1, 0, 64), (0, 64, 64)],
]


@pytest.mark.parametrize("H, Hkv", [(32, 4), (16, 16), (16, 1), (64, 32)])
@pytest.mark.parametrize("chunks", CHUNKS, ids=range(len(CHUNKS)))
def test_a_plan_lists_every_block_and_part(chunks, H, Hkv):
    both = ops.prefill_plan(chunks, H, Hkv, "cpu")
    one, other = ops.prefill_plan(chunks, H, Hkv, "cpu", kv8=False), ops.prefill_plan(chunks, H, Hkv, "cpu", kv8=True)
    assert one.kv8 is None and other.blocks is None
    rows = np.cumsum([0] + [n for *_, n in chunks])
    for p in (both, one, other):
        assert p.tables.T.tolist() == [[*c, int(r)] for c, r in zip(chunks, rows)]
        assert p.rows == rows[-1] and p.max_len == max([n for *_, n in chunks] + [0])
        assert p.pmax == max([1] + [(c + n - 1) // 6144 + 1 for _, c, n in chunks])
    for p in (both, one):
        assert p.blocks.is_contiguous() and [tuple(t) for t in p.blocks.T.tolist()] == _items(chunks, H, Hkv)
    for p in (both, other):
        assert p.kv8.tables.is_contiguous() and p.kv8.blocks.is_contiguous() and p.kv8.heads == (H, Hkv)
        assert torch.equal(p.kv8.tables, both.kv8.tables) and torch.equal(p.kv8.blocks, both.kv8.blocks)
        assert (p.kv8.units, p.kv8.slots) == (int(p.kv8.tables[0, -1]), int(p.kv8.tables[2, -1]))
        assert p.kv8.units == sum(-(-(c + n) // 64) for _, c, n in chunks)


def test_what_a_plan_refuses():
    for chunk in ((-1, 0, 1), (0, -1, 1), (0, 0, 0)):
        with pytest.raises(ValueError, match="chunk 1"):
            ops.prefill_plan([(0, 0, 5), chunk], 32, 4, "cpu")
    with pytest.raises(_lib.UnsupportedShape, match="H / Hkv"):
        ops.prefill_plan([(0, 0, 5)], 24, 8, "cpu", kv8=False)
    for chunk in ((0, 2 ** 32 + 5, 1), (2 ** 32, 0, 1)):  # (not what is left of it in 32 bits)
        with pytest.raises(OverflowError):
            ops.prefill_plan([chunk], 32, 4, "cpu")
    a, b, out = (np.array(x, np.int32) for x in ([0, 9], [5, 300], [0] * 99))
    call = lambda ctx, n, C=2, H=32, to=None, m=0: _lib.lib().jit_prefill_plan(  # noqa: E731
        ctx.ctypes.data if ctx is not None else None, n.ctypes.data if n is not None else None, C, H, 4,
        None if to is None else to.ctypes.data, m)
    n = call(a, b)
    assert n == len(_items([(0, 0, 5), (1, 9, 300)], 32, 4)) and call(a, b, to=out, m=n) == n and call(a, b, C=0) == 0
    assert call(a, b, to=out, m=n + 1) == call(a, b, to=out, m=n - 1) == call(None, b) == call(a, None) == EINVAL
    assert call(a, b, C=-1) == call(a, np.array([5, 0], np.int32)) == call(np.array([-1, 0], np.int32), b) == EINVAL
    assert call(np.array([0, 2 ** 31 - 1], np.int32), b) == EINVAL and call(a, b, H=24) == EUNSUPPORTED


@pytest.mark.gpu
def test_a_plan_serves_the_pools_that_it_is_made_for():
    H, Hkv, dev = 32, 4, "cuda"
    q = torch.randn((20, H, 128), generator=torch.Generator().manual_seed(1)).to(torch.bfloat16).to(dev)
    table = torch.arange(2, dtype=torch.int32, device=dev).view(1, 2)
    pool = torch.zeros((2, Hkv, 2, 2048), dtype=torch.bfloat16, device=dev)
    pool8 = ops.kv8_pool(2, Hkv, dev)
    k = torch.randn((32, Hkv, 128), generator=torch.Generator().manual_seed(2)).to(torch.bfloat16).to(dev)
    ops.kv8_append_paged(pool8, k, k, torch.arange(32, dtype=torch.int32, device=dev))
    plans = {kv8: ops.prefill_plan([(0, 12, 20)], H, Hkv, dev, kv8=kv8) for kv8 in (None, False, True)}
    run, run8 = ops.paged_prefill_attention, ops.paged_prefill_attention_kv8
    assert torch.equal(run(q, pool, table, plans[False], 0.1), run(q, pool, table, plans[None], 0.1))
    assert torch.equal(run8(q, pool8, table, plans[True], 0.1), run8(q, pool8, table, plans[None], 0.1))
    with pytest.raises(ValueError, match="no row blocks for a bf16 pool"):
        run(q, pool, table, plans[True], 0.1)
    with pytest.raises(ValueError, match="no row blocks for an 8-bit pool"):
        run8(q, pool8, table, plans[False], 0.1)


def test_the_registered_operator_refuses_tables_of_another_plan():
    """Its plan comes as tensors and numbers; what they are sized for has to be the chunks."""
    from jitengine_amd import torch_ops

    H, Hkv, chunks = 32, 4, [(0, 3000, 9), (1, 0, 400)]
    T = sum(n for *_, n in chunks)
    q, pool, table = torch.zeros((T, H, 128), dtype=torch.bfloat16), ops.kv8_pool(2, Hkv, "cpu"), torch.zeros((2, 200), dtype=torch.int32)
    plan = ops.prefill_plan(chunks, H, Hkv, "cpu")
    assert plan.kv8.slots > 0
    ws = torch.empty(16, dtype=torch.uint8)
    args = dict(zip(("tables", "chunk_tables", "blocks", "chunks", "units", "slots"), torch_ops.kv8_prefill_plan_args(plan)))
    call = lambda **other: torch.ops.jitengine.paged_prefill_attention_kv8(  # noqa: E731
        q, pool, table, *{**args, **other}.values(), 0.1, ws)
    ops.kv8_plan_contract(plan)
    with pytest.raises(ValueError, match="device tensor"):  # (the plan passes; the tensors here are the host's)
        call()
    for other in (
        {"units": plan.kv8.units + 1}, {"units": 1}, {"slots": 0}, {"slots": plan.kv8.slots - 1}, {"slots": -1},
        {"blocks": plan.kv8.blocks[:, :-1].contiguous()}, {"blocks": plan.kv8.blocks[:2].contiguous()},
        {"blocks": plan.blocks}, {"chunk_tables": plan.kv8.tables[:, :-1].contiguous()},
        {"chunk_tables": plan.tables}, {"tables": plan.tables[:, :1].contiguous()}, {"chunks": [0, 3000, 9]},
        {"chunks": [0, 3000, 9, 1, 0, 401]}, {"chunks": [0, 6000, 9, 1, 0, 400]}, {"chunks": []},
    ):
        with pytest.raises(ValueError, match="the plan's tables"):
            call(**other)
    with pytest.raises(ValueError, match="triples"):
        call(chunks=[0, 3000, 9, 1])
    with pytest.raises(ValueError):
        call(chunks=[0, 3000, 9, 1, 0, 0])
