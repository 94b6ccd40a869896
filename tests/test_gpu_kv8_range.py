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
    slots = (table[t // 16] * 16 + t % 16).int()
    for part in t.split(32768):  # (a write covers 65,535 rows)
        ops.kv8_append_paged(pool, k[part].to(DEV), v[part].to(DEV), slots[part].to(DEV))
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


@pytest.mark.parametrize("ctx, n", [(3000, 9), (0, 40)])
@pytest.mark.parametrize("mag", [2.0 ** -92, 1e-20])
def test_quiet_values_keep_their_bits_however_a_chunk_is_cut(ctx, n, mag):
    L, H, Hkv = ctx + n, 32, 4
    q, k, v = _normal(L, H, Hkv, n)
    q, k = (0.1 * q[:n]).to(torch.bfloat16), k.to(torch.bfloat16)
    v = ((1 + 0.05 * v.clamp(-1, 1)) * mag / 1.06).to(torch.bfloat16)
    pool, table = _cache(k, v)
    out, _ = _prompt(q.to(DEV), pool, table, ctx)
    want, A = _rows(q.to(DEV), pool, table, ctx)
    _check(out, want, A, 11, L, _score_error(q, k), (ctx, n, mag))


SHAPES = [(0, 2), (0, 70), (3000, 9), (20, 300), (8000, 16)]


@pytest.mark.parametrize("ctx, n", SHAPES)
@pytest.mark.parametrize("H, Hkv", [(32, 4), (16, 16)])
@pytest.mark.parametrize("power", [12, 13, 23, 40, 110])
def test_a_loud_value_leaves_the_rows_before_it_alone(ctx, n, H, Hkv, power):
    """The chunk's last token has V 2^power times its neighbours': the other rows do not see it."""
    L = ctx + n
    q, k, v = _normal(L, H, Hkv, n + power)
    q, k, v = q[:n].to(torch.bfloat16).to(DEV), k.to(torch.bfloat16), v.to(torch.bfloat16)
    v[-1] *= 2.0 ** power
    pool, table = _cache(k, v, power)
    out, _ = _prompt(q, pool, table, ctx)
    want, A = _rows(q, pool, table, ctx)
    _check(out, want, A, 11, L, _score_error(q, k), (ctx, n, power))


def test_a_quiet_first_row_is_its_own_value():
    """Two tokens, V of 1e-6 and then of 1e5: the first row gives its token's V as the cache holds it."""
    q, k, v = _normal(2, 8, 1, 5)
    k, v = k.to(torch.bfloat16), v.to(torch.bfloat16)
    v[0] *= 1e-6
    v[1] *= 1e5
    pool, table = _cache(k, v)
    out, _ = _prompt(q.to(torch.bfloat16).to(DEV), pool, table, 0)
    _, held = ref.read(pool, table[0].to(DEV))
    assert torch.equal(out[0].double(), held[0, :1].expand(8, 128))  # (4 significant bits: exact in bf16)


@pytest.mark.parametrize("ctx, n", [(0, 70), (3000, 9), (20, 300)])
@pytest.mark.parametrize("power", [-20, -40, -90])
def test_a_row_whose_weight_is_on_a_quiet_value(ctx, n, power):
    """Key 5 is 2^power as loud as the others and takes every row's weight but for some 2^-130."""
    H, Hkv, L = 32, 4, ctx + n
    q, k, v = _normal(L, H, Hkv, n)
    k = (k - 2 * k[5:6] * (k * k[5:6]).sum(-1, keepdim=True).clamp(min=0) / (k[5:6] ** 2).sum(-1, keepdim=True))
    k[5] = -k[5] / k[5].norm(dim=-1, keepdim=True) * 32  # (the others' products with it are zero or less)
    k = k.to(torch.bfloat16)
    q = (k[5].repeat_interleave(H // Hkv, 0)[None] * (1 + 0.01 * q[:n, :, :1])).to(torch.bfloat16).to(DEV)
    v = v.to(torch.bfloat16)
    v[5] *= 2.0 ** power
    pool, table = _cache(k, v, n)
    out, _ = _prompt(q, pool, table, ctx)
    want, A = _rows(q, pool, table, ctx)
    _check(out, want, A, 11, L, _score_error(q, k), (ctx, n, power))


@pytest.mark.parametrize("ctx, n", [(0, 70), (3000, 9), (40, 300)])
@pytest.mark.parametrize("power", [-8, -13, -30, -60, -85])
def test_quiet_values_beside_rows_of_zeros(ctx, n, power):
    """A block of zeros has scale 1, however quiet its neighbours are; slots that nothing was written to have scale 0."""
    H, Hkv, L = 32, 4, ctx + n
    q, k, v = _normal(L, H, Hkv, n)
    v *= 2.0 ** power
    v[torch.arange(0, L, 3)] = 0.0
    q, k = q[:n].to(torch.bfloat16).to(DEV), k.to(torch.bfloat16)
    pool, table = _cache(k, v.to(torch.bfloat16), n)
    pool[table[0, 1]] = 0
    out, _ = _prompt(q, pool, table, ctx)
    want, A = _rows(q, pool, table, ctx)
    _check(out, want, A, 11, L, _score_error(q, k), (ctx, n, power))


def test_parts_of_even_and_of_uneven_values_meet():
    """One of a chunk's 15 parts has values 2^30 louder than the others', with a weight that leaves both to be seen."""
    ctx, n, H, Hkv = 8000, 16, 32, 4
    L = ctx + n
    q, k, v = _normal(L, H, Hkv, 9)
    q, k, v = q[:n].to(torch.bfloat16).to(DEV), k.to(torch.bfloat16), v.to(torch.bfloat16)
    v[4000] *= 2.0 ** 16
    v[4001] *= 2.0 ** -14
    pool, table = _cache(k, v)
    out, plan = _prompt(q, pool, table, ctx)
    assert plan.kv8.slots >= 8 * n
    want, A = _rows(q, pool, table, ctx)
    _check(out, want, A, 11, L, _score_error(q, k), "parts")


def test_replays_over_even_and_uneven_values():
    """A captured chunk takes whatever values the cache holds when it is replayed."""
    ctx, n, H, Hkv = 640, 40, 32, 4
    L = ctx + n
    q, k, v = _normal(L, H, Hkv, 3)
    q, k, v = q[:n].to(torch.bfloat16).to(DEV), k.to(torch.bfloat16).to(DEV), v.to(torch.bfloat16).to(DEV)
    pool, table = _cache(k, v)
    t = table.int().to(DEV)
    at = torch.arange(L, device=DEV)
    slots = t[0, at // 16] * 16 + (at % 16).int()
    plan = ops.prefill_plan([(0, ctx, n)], H, Hkv, DEV)
    ws = torch.empty(ops.kv8_prefill_workspace_bytes(plan, H, Hkv), dtype=torch.uint8, device=DEV)
    ops.paged_prefill_attention_kv8(q, pool, t, plan, SCALE, ws)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = ops.paged_prefill_attention_kv8(q, pool, t, plan, SCALE, ws)
    for power in (0, 30, 0, -40, 5):
        v2 = v.clone()
        v2[L - 7] *= 2.0 ** power
        ops.kv8_append_paged(pool, k, v2, slots)
        graph.replay()
        torch.cuda.synchronize()
        want, A = _rows(q, pool, table, ctx)
        _check(out, want, A, 11, L, _score_error(q, k), power)
        eager = ops.paged_prefill_attention_kv8(q, pool, t, plan, SCALE)
        assert torch.equal(eager.view(torch.int16), out.view(torch.int16))


def _decode(q, k, v, seed, tag, pool_edit=None):
    """One sequence's single token over all of k, v, checked with 16 bits of a probability."""
    L = k.shape[0]
    pool, table = _cache(k, v, seed)
    if pool_edit:
        pool_edit(pool, table)
    t, n = table.int().to(DEV), torch.tensor([L], dtype=torch.int32, device=DEV)
    out = ops.paged_decode_attention_kv8(q, pool, t, n, L, SCALE)
    want, A = _rows(q, pool, table, L - 1)
    _check(out, want, A, 16, L, _score_error(q, k), tag)
    return out


@pytest.mark.parametrize("L", [1, 2, 33, 512, 513, 4096, 70001])
@pytest.mark.parametrize("H, Hkv", [(32, 4), (12, 4)])
def test_decode_keeps_16_bits_of_a_probability(L, H, Hkv):
    q, k, v = _normal(L, H, Hkv, L)
    _decode(q[:1].to(torch.bfloat16).to(DEV), k.to(torch.bfloat16), v.to(torch.bfloat16), L, L)


@pytest.mark.parametrize("L", [70, 600, 4100])
@pytest.mark.parametrize("power", [-8, -13, -30, -60, -85])
def test_decode_of_quiet_values_beside_rows_of_zeros(L, power):
    q, k, v = _normal(L, 32, 4, L)
    v *= 2.0 ** power
    v[torch.arange(0, L, 3)] = 0.0

    def empty_page(pool, table):
        pool[table[0, 1]] = 0
    _decode(q[:1].to(torch.bfloat16).to(DEV), k.to(torch.bfloat16), v.to(torch.bfloat16), L, (L, power), empty_page)


@pytest.mark.parametrize("L", [70, 4100, 40000])
@pytest.mark.parametrize("mag", [2.0 ** -92, 1e-20, 1e30, 1e36, 3e38])
def test_decode_of_even_values_of_any_magnitude(L, mag):
    """Sums of values, and of probabilities, that stay in fp32's range."""
    q, k, v = _normal(L, 32, 4, L)
    v = ((1 + 0.05 * v.clamp(-1, 1)) * (mag / 1.06)).to(torch.bfloat16)
    _decode((0.1 * q[:1]).to(torch.bfloat16).to(DEV), k.to(torch.bfloat16), v, L, (L, mag))


@pytest.mark.parametrize("L", [1, 40, 700])
@pytest.mark.parametrize("mag", [-1e30, -1e33, 1e33])
def test_decode_of_scores_of_any_magnitude(L, mag):
    """Keys that are all alike have the same weight, whatever their score."""
    q, k, v = _normal(L, 32, 4, L)
    k = torch.full((L, 4, 128), 2.0 ** 50).to(torch.bfloat16)
    q = torch.full((1, 32, 128), mag / 2.0 ** 50).to(torch.bfloat16).to(DEV)  # (scores about 11 mag)
    v = v.to(torch.bfloat16)
    pool, table = _cache(k, v, L)
    out = ops.paged_decode_attention_kv8(q, pool, table.int().to(DEV), torch.tensor([L], dtype=torch.int32, device=DEV), L, SCALE)
    _, held = ref.read(pool, table[0].to(DEV))
    held = held[:, :L].repeat_interleave(8, 0)
    _check(out, held.mean(1)[None], held.abs().mean(1)[None], 16, L, 0.0, (L, mag))


@pytest.mark.parametrize("power", [-90, -40, 40, 110])
def test_decode_of_one_value_far_from_the_others(power):
    L = 900
    q, k, v = _normal(L, 32, 4, 4)
    k, v = k.to(torch.bfloat16), v.to(torch.bfloat16)
    v[37] *= 2.0 ** power
    for on in (False, True):  # (with the weight on it, and as one of many)
        qq = (8 * k[37]).repeat_interleave(8, 0)[None] if on else q[:1].to(torch.bfloat16)
        _decode(qq.to(torch.bfloat16).to(DEV), k, v, 4, (power, on))


def test_rows_of_a_chunk_in_parts_are_those_of_a_larger_chunk():
    """16 rows after 8,000 keys are cut into parts, the same rows inside a chunk of 1,016 into others: the bits may
    differ, the values do not."""
    H, Hkv, L, n, more = 32, 4, 8016, 16, 1016
    q, k, v = _normal(L, H, Hkv, 6)
    q, k, v = q[:more].to(torch.bfloat16).to(DEV), k.to(torch.bfloat16), v.to(torch.bfloat16)
    pool, table = _cache(k, v)
    whole, wide = _prompt(q, pool, table, L - more)
    last, cut = _prompt(q[-n:].contiguous(), pool, table, L - n)
    assert int(cut.kv8.tables[1, 0]) != int(wide.kv8.tables[1, 0])  # (keys of a part)
    want, A = _rows(q[-n:], pool, table, L - n)
    for got in (last, whole[-n:]):
        _check(got, want, A, 11, L, _score_error(q, k), "cut")
