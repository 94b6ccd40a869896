"""The pool's handle of all layers: what it is made of, and when it is made anew (no GPU)."""

from __future__ import annotations

import torch

from jitengine_amd import ops
from jitengine_amd.kvpool import KVPool


def test_the_layers_handle_follows_the_pools_memory(monkeypatch):
    """Another tensor, the same tensor over other memory, a storage resized: each gives a handle of what is there now."""
    made = []
    monkeypatch.setattr(ops, "pool_layers", lambda pools: made.append([p.data_ptr() for p in pools]) or made[-1])
    pool = KVPool(3, 4, 1, "cpu")
    first = pool.layers()
    assert pool.layers() is first and len(made) == 1
    old = pool.pools[1].data
    pool.pools[1].data = old.clone()
    assert pool.layers() == [p.data_ptr() for p in pool.pools] != first
    pool.pools[2].set_(pool.pools[2].clone())
    assert pool.layers() == [p.data_ptr() for p in pool.pools]
    pool.pools = [p.clone() for p in pool.pools]
    assert pool.layers() == [p.data_ptr() for p in pool.pools] and len(made) == 4
    pool.pools[0].data = torch.zeros((8, 1, 2, 2048), dtype=torch.bfloat16)
    pool.layers()
    assert pool.layers() == [p.data_ptr() for p in pool.pools] and len(made) == 5


def test_layers_that_share_a_pool_have_it_once(monkeypatch):
    """Their pages were copied layer by layer before, the shared one as often as it stood there."""
    monkeypatch.setattr(ops, "pool_layers", list)
    pool = KVPool(4, 4, 1, "cpu")
    pool.pools[2] = pool.pools[0]
    assert [any(p is q for q in pool.layers()) for p in pool.pools] == [True] * 4 and len(pool.layers()) == 3
