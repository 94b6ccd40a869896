"""The 8-bit cache's attention over values of any magnitude that the cache holds (blocks' scales from 2^-100 to 2^118),
against its definition in 64 bits.  Tolerances are a row's own: keys that it does not see do not widen them."""

from __future__ import annotations

import math

import numpy as np
import pytest
import torch

from jitengine_amd import ops
from tests import kv8_ref as ref

pytestmark = pytest.mark.gpu
DEV = "cuda"
SCALE = 128 ** -0.5


def _i32(a) -> torch.Tensor:
    return torch.tensor(np.asarray(a), dtype=torch.int32).to(DEV)


def _cache(k: torch.Tensor, v: torch.Tensor, seed: int = 0, spare: int = 2):
    """k, v [n, Hkv, 128] bf16 as tokens 0 .. n - 1 of one sequence: (pool, table [1, W]); the rest of the pool's pages
    hold other tokens."""
    n, Hkv = k.shape[:2]
    W = -(-n // 16)
    table = torch.randperm(W + spare, generator=torch.Generator().manual_seed(seed + n))[:W]
    pool = ref.random_pool(W + spare, Hkv, seed + n, DEV)
    pool[table.to(DEV)] = 0
    t = torch.arange(n)
    ops.kv8_append_paged(pool, k.to(DEV), v.to(DEV), (table[t // 16] * 16 + t % 16).int().to(DEV))
    return pool, table.view(1, W)


def _rows(q, pool, table, ctx: int):
    """(out, sum p |v|) in 64 bits of q [n, H, 128]: row i sees the first ctx + i + 1 keys."""
    n, H, Hkv = q.shape[0], q.shape[1], pool.shape[1]
    G, L = H // Hkv, ctx + n
    k, v = ref.read(pool, table[0].to(DEV))
    k, v = k[:, :L], v[:, :L]
    hide = torch.arange(L, device=DEV)[None] > ctx + torch.arange(n, device=DEV)[:, None]
    out, A = [], []
    for h in range(Hkv):
        s = torch.einsum("ngd,kd->ngk", q[:, h * G:(h + 1) * G].double(), k[h]) * SCALE
        p = torch.softmax(s.masked_fill(hide[:, None], -math.inf), -1)
        out.append(torch.einsum("ngk,kd->ngd", p, v[h]))
        A.append(torch.einsum("ngk,kd->ngd", p, v[h].abs()))
    return torch.cat(out, 1), torch.cat(A, 1)


def _check(got, want, A, p_bits: int, n: int, ds: float, tag):
    """Half a bf16 step of the output; against sum p |v|: half a step of a probability's p_bits, one rounding of 2^-24
    a key of the fp32 sums on either side of the division, a score's error ds twice (numerator and denominator), and
    2^-20 for exp2 and the divisions.  Absolute: fp32's smallest normal number a key, over bf16's own."""
    tol = 2.0 ** -8 * want.abs() + (2.0 ** -p_bits + (n + 8) * 2.0 ** -23 + 2 * ds + 2.0 ** -20) * A + (n + 1) * 2.0 ** -126
    err = (got.double() - want).abs()
    bad = ~(err <= tol)
    assert not bool(bad.any()), (tag, int(bad.sum()), float((err / tol).nan_to_num(math.inf).max()), bad.nonzero()[0].tolist())


def _score_error(q, k) -> float:
    """A score's error: 2^-24 for each of 128 products and the scale, times the largest |q||k|."""
    return float(q.double().norm(dim=-1).max() * k.double().norm(dim=-1).max()) * SCALE * 130 * 2.0 ** -24


def _normal(n, H, Hkv, seed):
    g = torch.Generator().manual_seed(seed)
    r = lambda *s: torch.randn(s, generator=g)
    return r(n, H, 128), r(n, Hkv, 128), r(n, Hkv, 128)


def _prompt(q, pool, table, ctx):
    n, H = q.shape[:2]
    plan = ops.prefill_plan([(0, ctx, n)], H, pool.shape[1], DEV)
    return ops.paged_prefill_attention_kv8(q, pool, table.int().to(DEV), plan, SCALE), plan


@pytest.mark.parametrize("ctx, n", [(3000, 9), (0, 40)])
@pytest.mark.parametrize("mag", [1e30, 1e36, 3e38])
def test_loud_values_stay_finite_however_a_chunk_is_cut(ctx, n, mag):
    """Even values near bf16's largest: a mean of them is as large, a sum of them is not a number of fp32."""
    L, H, Hkv = ctx + n, 32, 4
    q, k, v = _normal(L, H, Hkv, n)
    q, k = (0.1 * q[:n]).to(torch.bfloat16), k.to(torch.bfloat16)  # (scores of about 0.1: every key counts)
    v = ((1 + 0.05 * v.clamp(-1, 1)) * mag / 1.06).to(torch.bfloat16)
    assert bool(v.isfinite().all())
    pool, table = _cache(k, v)
    out, plan = _prompt(q.to(DEV), pool, table, ctx)
    assert (plan.kv8.slots > 0) == (ctx > 0)
    want, A = _rows(q.to(DEV), pool, table, ctx)
    _check(out, want, A, 11, L, _score_error(q, k), (ctx, n, mag))
