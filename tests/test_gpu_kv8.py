"""The 8-bit KV cache on the GPU against its restatement in 64 bits (tests/kv8_ref.py): the bytes a write leaves,
attention of single tokens and of prompt chunks where masks, pages and lengths can go wrong, a step's tables, and the
calls of a step in a row."""

from __future__ import annotations

import random

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


def _bits(t):
    return t.view(torch.int16)


def _same_bytes(got, want):
    off = (got != want).nonzero()
    assert not len(off), [(*p, int(got[tuple(p)]), int(want[tuple(p)])) for p in off[:8].tolist()] + [len(off)]


def _special(g, B, Hkv) -> torch.Tensor:
    """bf16 rows [B, Hkv, 128] of every magnitude a block can have."""
    x = torch.randn((B, Hkv, 128), generator=g)
    x[0] = 0.0
    x[1] *= 1e38
    x[2] *= 1e-38
    x[3, 0, 5], x[3, 0, 77], x[3, 0, 100] = float("nan"), float("inf"), -float("inf")
    x[4, 0] = 0.25
    x[4, 0, 64] = 1.75          # the largest value that keeps its exponent
    x[5, 0] = 0.25
    x[5, 0, 63] = 1.765625      # the next bf16: one exponent up
    x[6, 0] = 3.3895313892515355e38
    x[7, 0] = 0.0
    x[7, 0, 127] = -2.0 ** -133
    return x.to(torch.bfloat16)


@pytest.mark.parametrize("B, Hkv", [(1, 1), (9, 4), (40, 2), (33, 16), (257, 3)])
def test_append_leaves_the_defined_bytes(B, Hkv):
    g = torch.Generator().manual_seed(B)
    k, v = torch.randn((B, Hkv, 128), generator=g).to(torch.bfloat16), torch.randn((B, Hkv, 128), generator=g).to(torch.bfloat16)
    if B >= 9:
        k, v = _special(g, B, Hkv), _special(g, B, Hkv).flip(0)
    pages = B // 8 + 2
    pool = ref.random_pool(pages, Hkv, B)
    slots = torch.randperm(pages * 16, generator=g)[:B].to(torch.int32)
    if B > 20:  # rows that are not written
        slots[10], slots[11], slots[12], slots[13] = -1, pages * 16, 2 ** 31 - 1, -(2 ** 31)
    got = pool.to(DEV)
    ops.kv8_append_paged(got, k.to(DEV), v.to(DEV), slots.to(DEV))
    ref.write(pool, k, v, slots)
    _same_bytes(got.cpu(), pool)


@pytest.mark.parametrize("n, slot0", [(16, 0), (47, 5), (64, 30), (1, 15), (130, 16)])
def test_append_of_consecutive_slots(n, slot0):
    """Prompt rows fill pages in order, from the middle of one to the middle of another, in permuted pages."""
    g = torch.Generator().manual_seed(n)
    Hkv, pages = 4, (slot0 + n) // 16 + 2
    k, v = (torch.randn((n, Hkv, 128), generator=g).to(torch.bfloat16) for _ in range(2))
    perm = torch.randperm(pages, generator=g)
    at = slot0 + torch.arange(n)
    slots = (perm[at // 16] * 16 + at % 16).to(torch.int32)
    pool = ref.random_pool(pages, Hkv, n)
    got = pool.to(DEV)
    ops.kv8_append_paged(got, k.to(DEV), v.to(DEV), slots.to(DEV))
    ref.write(pool, k, v, slots)
    _same_bytes(got.cpu(), pool)


def _norm_rope(x, w, eps, pos, inv_freq):
    x, w = x.double(), w.double()
    y = x / torch.sqrt((x * x).mean(-1, keepdim=True) + eps) * w
    ang = (pos.double()[:, None] * inv_freq.double())[:, None]
    c, s = torch.cos(ang), torch.sin(ang)
    a, b = y[..., :64], y[..., 64:]
    return torch.cat([a * c - b * s, a * s + b * c], -1)


@pytest.mark.parametrize("B, H, Hkv, top", [(1, 32, 4, 4096), (32, 32, 4, 262144), (70, 8, 8, 50), (19, 64, 4, 2 ** 31 - 1),
                                            (333, 12, 4, 8192)])
def test_norm_rope_append(B, H, Hkv, top):
    g = torch.Generator().manual_seed(B + H)
    qkv = (2 * torch.randn((B, (H + 2 * Hkv) * 128), generator=g)).to(torch.bfloat16)
    qw, kw = ((1 + 0.3 * torch.randn(128, generator=g)).to(torch.bfloat16) for _ in range(2))
    inv = torch.from_numpy((1e6 ** (-np.arange(0, 128, 2) / 128)).astype(np.float32))
    pos = torch.randint(0, top, (B,), generator=g)
    pos[0] = top - 1
    pages = B // 8 + 2
    slots = torch.randperm(pages * 16, generator=g)[:B].to(torch.int32)
    if B > 3:
        slots[2] = -1  # (its q is made all the same)
    pool = ref.random_pool(pages, Hkv, 5)
    got = pool.to(DEV)
    q = ops.qk_norm_rope_append_kv8(qkv.to(DEV), H, Hkv, qw.to(DEV), kw.to(DEV), 1e-6, inv.to(DEV), pos.to(torch.int32).to(DEV),
                                    slots.to(DEV), got).cpu()
    got = got.cpu()
    x = qkv.view(B, H + 2 * Hkv, 128)
    want = _norm_rope(x[:, :H], qw, 1e-6, pos, inv)
    # half a bf16 step; fp32 products, sums, rsqrt and sincos before it: a dozen roundings of the pair's magnitude
    pair = torch.hypot(want[..., :64], want[..., 64:]).repeat(1, 1, 2)
    assert bool(((q.double() - want).abs() <= 2.0 ** -8 * want.abs() + 12 * 2.0 ** -23 * pair + 2.0 ** -133).all())
    k, v = _norm_rope(x[:, H:H + Hkv], kw, 1e-6, pos, inv), x[:, H + Hkv:].double()
    pair = torch.hypot(k[..., :64], k[..., 64:]).repeat(1, 1, 2)
    (_, ke), (vc, ve) = ref.quantise(k), ref.quantise(v)
    lut, d, sc = ref.e4m3_values(), torch.arange(128), ref.scales(got)
    others = torch.ones(pages * 16, dtype=torch.bool)
    for b, s in enumerate(slots.tolist()):
        if s < 0:
            continue
        others[s] = False
        p, t = divmod(s, 16)
        assert torch.equal(got[p][:, ref.v_at(t, d)].long(), vc[b])
        assert torch.equal(sc[p, :, 16 + t].double(), torch.exp2(ve[b].double()))
        gs = sc[p, :, t].double()
        # the scale is that of the exact block, or its neighbour where fp32 may see the largest on the other side
        amax = k[b].abs().amax(-1)
        lo, hi = ref.scale_exp(amax * (1 - 2.0 ** -19)), ref.scale_exp(amax * (1 + 2.0 ** -19))
        e = torch.log2(gs)
        assert bool(((e == lo) | (e == hi)).all())
        back = lut[got[p][:, ref.k_at(t, d)].long()] * gs[:, None]
        # half an e4m3 step of the value or of the smallest one, and fp32's part as for q
        tol = torch.maximum(2.0 ** -4 * k[b].abs(), gs[:, None] * 2.0 ** -10) + 12 * 2.0 ** -23 * pair[b]
        assert bool(((back - k[b]).abs() <= tol).all())
    # every other slot keeps its bytes
    t = torch.arange(16)
    keep = others.view(pages, 16)
    for p in range(pages):
        for s in t[keep[p]].tolist():
            for at in (ref.k_at(s, d), ref.v_at(s, d)):
                assert torch.equal(got[p][:, at], pool[p][:, at])
            assert torch.equal(sc[p, :, [s, 16 + s]], ref.scales(pool)[p, :, [s, 16 + s]])


def _table(lens, seed, extra=2):
    """(page table [B, W], pages) over permuted pages; entries past a sequence's pages point outside the pool."""
    rng = np.random.default_rng(seed)
    npg = [-(-n // 16) for n in lens]
    total = sum(npg) + extra
    perm = rng.permutation(total)
    t = np.full((len(lens), max(npg + [1])), 2 ** 31 - 1, np.int64)
    at = 0
    for i, n in enumerate(npg):
        t[i, :n] = perm[at:at + n]
        at += n
    return t, total


def _poison_stale(pool, table, lens):
    """NaN codes and wild scales in every slot past a sequence's length (what a recycled page may hold)."""
    sc, d = ref.scales(pool), torch.arange(128, device=pool.device)
    for b, n in enumerate(lens):
        if n % 16:
            p = int(table[b, n // 16])
            for s in range(n % 16, 16):
                pool[p][:, ref.k_at(s, d)] = 127
                pool[p][:, ref.v_at(s, d)] = 255
                sc[p, :, s] = float("nan")
                sc[p, :, 16 + s] = float("inf") if s % 2 else float("nan")


def _check_decode(out, q, pool, table, lens, tag):
    B, H, _ = q.shape
    Hkv = pool.shape[1]
    G = H // Hkv
    for b, n in enumerate(lens):
        if n == 0:
            assert not bool(out[b].any())
            continue
        k, v = ref.read(pool, table[b, :-(-n // 16)])
        for h in range(Hkv):
            want, tol = ref.attend(q[b:b + 1, h * G:(h + 1) * G], k[h, :n], v[h, :n], SCALE)
            err = (out[b:b + 1, h * G:(h + 1) * G].double() - want).abs()
            assert bool((err <= tol).all()), (tag, b, n, h, float((err - tol).max()), float((err / tol).max()))


LENS = [1, 2, 15, 16, 17, 31, 32, 33, 64, 127, 128, 129, 511, 512, 513, 700, 2049, 0]


@pytest.mark.parametrize("H, Hkv", [(32, 4), (16, 16), (64, 4), (12, 4), (8, 1), (3, 3)])
def test_decode_attention(H, Hkv):
    g = torch.Generator().manual_seed(H)
    table, pages = _table(LENS, H)
    pool = ref.random_pool(pages, Hkv, H, DEV, v_spread=2.0)
    _poison_stale(pool, table, LENS)
    q = (1.5 * torch.randn((len(LENS), H, 128), generator=g)).to(torch.bfloat16).to(DEV)
    out = ops.paged_decode_attention_kv8(q, pool, _i32(table), _i32(LENS), max(LENS), SCALE)
    _check_decode(out, q, pool, torch.from_numpy(table).to(DEV), LENS, (H, Hkv))


@pytest.mark.parametrize("n", [65536, 65537, 100003, 200001])
def test_decode_attention_of_long_sequences(n):
    lens = [n, 40]
    table, pages = _table(lens, n)
    pool = ref.random_pool(pages, 2, 3, DEV)
    _poison_stale(pool, table, lens)
    q = torch.randn((2, 16, 128), generator=torch.Generator().manual_seed(n)).to(torch.bfloat16).to(DEV)
    out = ops.paged_decode_attention_kv8(q, pool, _i32(table), _i32(lens), n, SCALE)
    _check_decode(out, q, pool, torch.from_numpy(table).to(DEV), lens, n)


def test_a_decode_row_does_not_depend_on_its_batch_or_bound():
    lens = [700, 3, 5000, 513, 1, 20000, 16, 1030]
    table, pages = _table(lens, 4)
    pool = ref.random_pool(pages, 4, 4, DEV)
    t = _i32(table)
    q = torch.randn((len(lens), 32, 128), generator=torch.Generator().manual_seed(4)).to(torch.bfloat16).to(DEV)
    out = ops.paged_decode_attention_kv8(q, pool, t, _i32(lens), max(lens), SCALE)
    for b, n in enumerate(lens):
        for most in {n, max(lens)}:
            one = ops.paged_decode_attention_kv8(q[b:b + 1], pool, t[b:b + 1].contiguous(), _i32([n]), most, SCALE)
            assert torch.equal(_bits(one[0]), _bits(out[b])), (b, n, most)
    many = ops.paged_decode_attention_kv8(q.repeat(40, 1, 1), pool, t.repeat(40, 1), _i32(lens * 40), max(lens), SCALE)
    assert torch.equal(_bits(many), _bits(out.repeat(40, 1, 1)))
    # a bound below a length cuts the sequence there
    cut = ops.paged_decode_attention_kv8(q, pool, t, _i32(lens), 513, SCALE)
    want = ops.paged_decode_attention_kv8(q, pool, t, _i32([min(n, 513) for n in lens]), 513, SCALE)
    assert torch.equal(_bits(cut), _bits(want))
    neg = ops.paged_decode_attention_kv8(q, pool, t, _i32([-5] * len(lens)), 64, SCALE)
    assert not bool(neg.any())


def test_decode_leaves_out_pages_outside_the_pool():
    n = 700
    table, pages = _table([n, n], 6)
    table[0, 3], table[0, 10], table[0, 43], table[0, 0] = -1, pages, -(2 ** 31), 2 ** 31 - 1
    keep = torch.ones(n, dtype=torch.bool)
    for p in (0, 3, 10, 43):
        keep[16 * p:16 * p + 16] = False
    table[1, :] = -7  # no key at all
    pool = ref.random_pool(pages, 4, 6, DEV)
    q = torch.randn((2, 32, 128), generator=torch.Generator().manual_seed(6)).to(torch.bfloat16).to(DEV)
    out = ops.paged_decode_attention_kv8(q, pool, _i32(table), _i32([n, n]), n, SCALE)
    assert not bool(out[1].any())
    rows = torch.from_numpy(np.where((table[0] < 0) | (table[0] >= pages), 0, table[0]))
    k, v = ref.read(pool, rows)
    for h in range(4):
        want, tol = ref.attend(q[:1, 8 * h:8 * h + 8], k[h, :n], v[h, :n], SCALE, keep[None].to(DEV))
        assert bool(((out[:1, 8 * h:8 * h + 8].double() - want).abs() <= tol).all())


def test_decode_of_uneven_values_and_empty_slots():
    """A key with nearly all of the weight and tiny values beside loud ones with little weight, a q that is not
    finite, and live slots of a page that nothing was written to (zeros)."""
    lens = [300, 300, 64, 300]
    table, pages = _table(lens, 8)
    pool = ref.random_pool(pages, 4, 8, DEV)
    t = torch.from_numpy(table).to(DEV)
    p0 = int(table[0, 2])
    ref.scales(pool)[p0, :, 16 + 5] = 2.0 ** -90   # key 37 of sequence 0
    ref.scales(pool)[int(table[1, 7]), :, 16 + 1] = 2.0 ** 40
    for i in range(4):
        pool[int(table[2, i])] = 0
    q = torch.randn((4, 32, 128), generator=torch.Generator().manual_seed(8)).to(torch.bfloat16).to(DEV)
    k, _ = ref.read(pool, t[0, :19])
    q[0] = (k[:, 37] * 8).repeat_interleave(8, 0).to(torch.bfloat16)  # key 37 takes the weight
    q[3, 5, 3] = float("nan")
    out = ops.paged_decode_attention_kv8(q, pool, t.int(), _i32(lens), 300, SCALE)
    _check_decode(out[:2], q[:2], pool, t, lens[:2], "uneven")
    assert not bool(out[2].any())
    assert bool(torch.isnan(out[3, 5]).all()) and bool(torch.isfinite(out[3, :5]).all()) and bool(torch.isfinite(out[3, 6:]).all())


def _check_prefill(out, q, pool, table, chunks, tag, bad=()):
    H, Hkv = q.shape[1], pool.shape[1]
    G, row = H // Hkv, 0
    for c, (seq, ctx, n) in enumerate(chunks):
        keys = ctx + n
        pg = table[seq, :-(-keys // 16)]
        ok = (pg >= 0) & (pg < pool.shape[0])
        k, v = ref.read(pool, torch.where(ok, pg, torch.zeros_like(pg)))
        keep = torch.arange(keys, device=DEV)[None] <= ctx + torch.arange(n, device=DEV)[:, None]
        keep &= ok.repeat_interleave(16)[:keys][None]
        for h in range(Hkv):
            want, tol = ref.attend(q[row:row + n, h * G:(h + 1) * G], k[h, :keys], v[h, :keys], SCALE, keep)
            err = (out[row:row + n, h * G:(h + 1) * G].double() - want).abs()
            assert bool((err <= tol).all()), (tag, c, h, float((err / tol).max()))
        row += n


CHUNKS = {
    "one_token": [(0, 0, 1)],
    "short": [(0, 0, 5), (1, 3, 1), (2, 16, 15), (3, 0, 16), (4, 127, 2), (5, 250, 17)],
    "odd": [(0, 0, 77)],
    "blocks": [(0, 100, 33), (1, 0, 65), (2, 31, 300)],
    "shared": [(0, 0, 40), (0, 40, 24), (0, 64, 9)],  # three chunks of one sequence
    "parts": [(0, 6140, 9), (1, 6100, 40), (2, 12280, 30), (3, 5, 3)],
}


@pytest.mark.parametrize("H, Hkv", [(32, 4), (16, 16), (16, 1), (8, 4)])
@pytest.mark.parametrize("name", list(CHUNKS))
def test_prefill_attention(name, H, Hkv):
    chunks = CHUNKS[name]
    S = max(s for s, _, _ in chunks) + 1
    lens = [max([c + n for s, c, n in chunks if s == i] + [0]) for i in range(S)]
    table, pages = _table(lens, len(name))
    pool = ref.random_pool(pages, Hkv, len(name), DEV, v_spread=2.0)
    _poison_stale(pool, table, lens)
    T = sum(n for _, _, n in chunks)
    q = (1.5 * torch.randn((T, H, 128), generator=torch.Generator().manual_seed(T))).to(torch.bfloat16).to(DEV)
    out = ops.paged_prefill_attention_kv8(q, pool, _i32(table), ops.prefill_plan(chunks, H, Hkv, DEV), SCALE)
    _check_prefill(out, q, pool, torch.from_numpy(table).to(DEV), chunks, name)


def test_prefill_of_many_row_blocks():
    """Enough work items for whole row blocks a workgroup (each rule of the launch)."""
    for n_chunk, n in ((1, 600), (3, 500), (9, 310)):
        chunks = [(i, 17 * i, n) for i in range(n_chunk)]
        lens = [c + m for _, c, m in chunks]
        table, pages = _table(lens, n)
        pool = ref.random_pool(pages, 8, n, DEV)
        q = torch.randn((n * n_chunk, 32, 128), generator=torch.Generator().manual_seed(n)).to(torch.bfloat16).to(DEV)
        out = ops.paged_prefill_attention_kv8(q, pool, _i32(table), ops.prefill_plan(chunks, 32, 8, DEV), SCALE)
        _check_prefill(out, q, pool, torch.from_numpy(table).to(DEV), chunks, n)


def test_a_prompt_row_does_not_depend_on_the_cut():
    n = 333
    table, pages = _table([n], 3)
    pool = ref.random_pool(pages, 4, 3, DEV)
    t = _i32(table)
    q = torch.randn((n, 32, 128), generator=torch.Generator().manual_seed(3)).to(torch.bfloat16).to(DEV)
    whole = ops.paged_prefill_attention_kv8(q, pool, t, ops.prefill_plan([(0, 0, n)], 32, 4, DEV), SCALE)
    at = 0
    for m in (1, 31, 100, 16, 150, 35):
        part = ops.paged_prefill_attention_kv8(q[at:at + m].contiguous(), pool, t,
                                               ops.prefill_plan([(0, at, m)], 32, 4, DEV), SCALE)
        assert torch.equal(_bits(part), _bits(whole[at:at + m])), m
        at += m


def test_prefill_leaves_out_pages_outside_the_pool_and_takes_uneven_values():
    chunks = [(0, 200, 70), (1, 0, 20), (2, 0, 200)]
    lens = [270, 20, 200]
    table, pages = _table(lens, 9)
    table[0, 2], table[0, 9], table[0, 16] = -1, pages, 2 ** 31 - 1
    table[1, 0] = -3  # rows 0 .. 15 of chunk 1 see no key
    pool = ref.random_pool(pages, 4, 9, DEV)
    sc = ref.scales(pool)
    sc[int(table[2, 1]), :, 16 + 3] = 2.0 ** -20
    sc[int(table[2, 9]), :, 16 + 2] = 2.0 ** 9   # louder values in the second step
    q = torch.randn((290, 32, 128), generator=torch.Generator().manual_seed(9)).to(torch.bfloat16).to(DEV)
    out = ops.paged_prefill_attention_kv8(q, pool, _i32(table), ops.prefill_plan(chunks, 32, 4, DEV), SCALE)
    _check_prefill(out, q, pool, torch.from_numpy(table).to(DEV), chunks, "bad")
    assert not bool(out[70:86].any())


def _check_tables(ctx, new, table, rows, free=None, free_at=None):
    t = _i32(table) if len(table) else torch.zeros((0, 3), dtype=torch.int32, device=DEV)
    got = ops.step_tables(_i32(ctx), _i32(new), t, rows, free=None if free is None else _i32(free),
                          free_at=None if free_at is None else _i32([free_at]))
    grown = [list(map(int, r)) for r in table]
    want = ref.step_tables(ctx, new, grown, rows, free, free_at or 0)
    for name, w in want.items():
        assert getattr(got, name).tolist() == w, name
    assert t.tolist() == grown
    return got


@pytest.mark.parametrize("seed", range(12))
def test_step_tables(seed):
    r = random.Random(seed)
    S = r.choice([1, 2, 7, 64, 300, 1500])
    W = r.choice([4, 20, 70])
    ctx = [r.randint(0, 15 * W) for _ in range(S)]
    new = [r.choice([0, 1, 1, 1, r.randint(0, 40)]) for _ in range(S)]
    perm = r.sample(range(S * W + 50), S * W + 50)
    table = [[perm.pop() if j < -(-c // 16) else -1 for j in range(W)] for c in ctx]
    need = sum(-(-(c + n) // 16) - -(-c // 16) for c, n in zip(ctx, new))
    rows = max(0, sum(new) + r.choice([0, 0, 5, -3]))
    for have in (need + 3, need, need // 2, 0):
        _check_tables(ctx, new, table, rows, perm[:have + 2], 2 if seed % 2 else None)
    full = [[x if x >= 0 else 7 for x in row] for row in table]
    _check_tables(ctx, new, full, rows)


def test_step_tables_at_the_edges():
    _check_tables([], [], [], 5)
    _check_tables([], [], [], 0)
    _check_tables([0], [0], [[5, 6]], 0)
    _check_tables([-3, 2 ** 31 - 1, 5], [4, 2 ** 31 - 1, -9], [[1, 2], [3, 4], [5, 6]], 6)   # values no step has
    _check_tables([31], [2], [[1, 2]], 2, [9, 8])                                            # past the table's width
    _check_tables([16, 16], [1, 1], [[1, -5], [2, 1 << 27]], 2)                              # ids no slot can have
    _check_tables([0] * 8192, [1] * 8192, [[i] for i in range(8192)], 8192)
    _check_tables([3] * 5, [20, 0, 5, 13, 14], [[i, -1, -1] for i in range(5)], 60, list(range(100, 104)))


@pytest.mark.parametrize("Hkv", [1, 4])
def test_copy_pages(Hkv):
    pool = ref.random_pool(9, Hkv, 1)
    got = pool.to(DEV)
    ops.kv8_copy_pages(got, _i32([3, 0, -1, 2, 99]), _i32([7, 8, 1, 9, 4]))
    pool[7], pool[8] = pool[3], pool[0]
    _same_bytes(got.cpu(), pool)


def _step_inputs(S, H, Hkv, W, seed):
    g = torch.Generator().manual_seed(seed)
    inv = torch.from_numpy((1e6 ** (-np.arange(0, 128, 2) / 128)).astype(np.float32)).to(DEV)
    w = [(1 + 0.1 * torch.randn(128, generator=g)).to(torch.bfloat16).to(DEV) for _ in range(2)]
    qkv = [torch.randn((S, (H + 2 * Hkv) * 128), generator=g).to(torch.bfloat16).to(DEV) for _ in range(40)]
    return inv, w, qkv


def test_steps_in_a_row_eager_and_replayed():
    """Tables, write and attention of decode steps whose lengths and tables live on the device: eager against the
    restatement, and the same steps replayed from one captured graph, with eager work in between."""
    S, H, Hkv, W = 5, 16, 4, 8
    start = [0, 15, 16, 30, 47]
    inv, w, qkv = _step_inputs(S, H, Hkv, W, 1)
    free = _i32(list(np.random.default_rng(1).permutation(40)))

    class Run:
        def __init__(self):
            self.pool = ops.kv8_pool(48, Hkv, DEV)
            self.table = torch.full((S, W), -1, dtype=torch.int32, device=DEV)
            for b, n in enumerate(start):  # the pages of what is there already
                for j in range(-(-n // 16)):
                    self.table[b, j] = 40 + b
            self.ctx, self.at, self.new = _i32(start), _i32([0]), _i32([1] * S)
            self.x = qkv[0].clone()

        def step(self):
            t = ops.step_tables(self.ctx, self.new, self.table, S, free=free, free_at=self.at)
            q = ops.qk_norm_rope_append_kv8(self.x, H, Hkv, w[0], w[1], 1e-6, inv, t.pos, t.slots, self.pool)
            out = ops.paged_decode_attention_kv8(q, self.pool, self.table, t.lens, 16 * W, SCALE)
            self.ctx.copy_(t.lens)
            self.at.copy_(t.status[1:2])
            return q, out

    a, b = Run(), Run()
    a.step()  # (warm; both runs start over below)
    a = Run()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        gq, gout = b.step()
    b.ctx.copy_(_i32(start))
    b.at.zero_()
    for i in range(30):
        a.x.copy_(qkv[i])
        b.x.copy_(qkv[i])
        q, out = a.step()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(_bits(gq), _bits(q)) and torch.equal(_bits(gout), _bits(out)), i
        lens = [n + i + 1 for n in start]
        assert a.ctx.tolist() == lens and b.ctx.tolist() == lens
        assert torch.equal(a.pool, b.pool) and torch.equal(a.table, b.table)
        if i % 7 == 0:
            _check_decode(out, q, a.pool, a.table, lens, i)


def test_calls_on_two_streams_share_nothing():
    lens = [3000, 17]
    table, pages = _table(lens, 2)
    pool = ref.random_pool(pages, 4, 2, DEV)
    t, n = _i32(table), _i32(lens)
    qs = [torch.randn((2, 32, 128), generator=torch.Generator().manual_seed(i)).to(torch.bfloat16).to(DEV) for i in range(2)]
    want = [ops.paged_decode_attention_kv8(q, pool, t, n, 3000, SCALE) for q in qs]
    ws = [torch.empty(ops.kv8_decode_workspace_bytes(2, 32, 3000), dtype=torch.uint8, device=DEV) for _ in range(2)]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = []
    for _ in range(10):
        for q, s, m in zip(qs, streams, ws):
            with torch.cuda.stream(s):
                got.append(ops.paged_decode_attention_kv8(q, pool, t, n, 3000, SCALE, m))
    torch.cuda.synchronize()
    for i, o in enumerate(got):
        assert torch.equal(_bits(o), _bits(want[i % 2]))


def test_refusals_on_device_tensors():
    pool = ops.kv8_pool(8, 4, DEV)
    i = _i32([0, 1])
    t = torch.zeros((2, 4), dtype=torch.int32, device=DEV)
    kv = torch.zeros((2, 4, 128), dtype=torch.bfloat16, device=DEV)
    q = torch.zeros((2, 32, 128), dtype=torch.bfloat16, device=DEV)
    qkv = torch.zeros((2, 40 * 128), dtype=torch.bfloat16, device=DEV)
    w = torch.zeros(128, dtype=torch.bfloat16, device=DEV)
    f = torch.zeros(64, device=DEV)
    plan = ops.prefill_plan([(0, 0, 2)], 32, 4, DEV)
    bad = [
        lambda: ops.kv8_append_paged(pool[:, :2], kv, kv, i),
        lambda: ops.kv8_append_paged(pool.bfloat16(), kv, kv, i),
        lambda: ops.kv8_append_paged(pool, kv[:, :2].contiguous(), kv, i),
        lambda: ops.kv8_append_paged(pool, kv, kv.transpose(0, 1), i),
        lambda: ops.kv8_append_paged(pool, kv, kv, i.long()),
        lambda: ops.kv8_append_paged(pool, kv, kv, i.cpu()),
        lambda: ops.kv8_append_paged(pool, kv, kv, i[:1]),
        lambda: ops.qk_norm_rope_append_kv8(qkv, 32, 2, w, w, 1e-6, f, i, i, pool),
        lambda: ops.qk_norm_rope_append_kv8(qkv, 32, 4, w[:64], w, 1e-6, f, i, i, pool),
        lambda: ops.qk_norm_rope_append_kv8(qkv, 32, 4, w, w, 1e-6, f.double(), i, i, pool),
        lambda: ops.qk_norm_rope_append_kv8(qkv, 32, 4, w, w, 1e-6, f, i[:1], i, pool),
        lambda: ops.paged_decode_attention_kv8(q, pool, t, i[:1], 64, SCALE),
        lambda: ops.paged_decode_attention_kv8(q, pool, t, i, 65, SCALE),
        lambda: ops.paged_decode_attention_kv8(q, pool, t, i, -1, SCALE),
        lambda: ops.paged_decode_attention_kv8(q[:, :30].contiguous(), pool, t, i, 64, SCALE),
        lambda: ops.paged_decode_attention_kv8(q.view(4, 32, 64), pool, t, i, 64, SCALE),
        lambda: ops.paged_decode_attention_kv8(q.float(), pool, t, i, 64, SCALE),
        lambda: ops.paged_prefill_attention_kv8(q[:1], pool, t, plan, SCALE),
        lambda: ops.paged_prefill_attention_kv8(q, pool, t[:, :0].contiguous(), plan, SCALE),
        lambda: ops.step_tables(i, i[:1], t, 2),
        lambda: ops.step_tables(i, i, t[:1], 2),
        lambda: ops.step_tables(i, i, t, -1),
        lambda: ops.step_tables(i, i, t, 2, free_at=i[:1]),
        lambda: ops.step_tables(i, i, t.t(), 2),
        lambda: ops.step_tables(i.long(), i, t, 2),
        lambda: ops.kv8_copy_pages(pool, i, i[:1]),
        lambda: ops.kv8_copy_pages(pool, i.long(), i.long()),
    ]
    for n, call in enumerate(bad):
        with pytest.raises(ValueError):
            call()
            pytest.fail(f"call {n} was taken")
    # no rows: nothing to do
    assert ops.paged_decode_attention_kv8(q[:0], pool, t[:0], i[:0], 64, SCALE).shape == (0, 32, 128)
    ops.kv8_append_paged(pool, kv[:0], kv[:0], i[:0])
    assert not bool(pool.any())


@pytest.mark.parametrize("H, Hkv", [(32, 4), (128, 16), (16, 16)])
def test_a_chunk_of_many_key_parts_does_not_depend_on_its_call(H, Hkv):
    """Few rows after many keys are cut into many parts; a chunk's bits are those of the chunk alone."""
    chunks = [(0, 3000, 9), (1, 0, 400), (2, 5001, 1), (3, 640, 130)]
    lens = [c + n for _, c, n in chunks]
    table, pages = _table(lens, H)
    pool = ref.random_pool(pages, Hkv, H, DEV, v_spread=2.0)
    _poison_stale(pool, table, lens)
    t, T = _i32(table), sum(n for *_, n in chunks)
    plan = ops.prefill_plan(chunks, H, Hkv, DEV)
    assert plan.kv8.slots > 0 and int(plan.kv8.blocks[2].max()) >= 4
    q = torch.randn((T, H, 128), generator=torch.Generator().manual_seed(H)).to(torch.bfloat16).to(DEV)
    out = ops.paged_prefill_attention_kv8(q, pool, t, plan, SCALE)
    _check_prefill(out, q, pool, torch.from_numpy(table).to(DEV), chunks, (H, Hkv))
    row = 0
    for s, c, n in chunks:
        alone = ops.paged_prefill_attention_kv8(q[row:row + n].contiguous(), pool, t,
                                                ops.prefill_plan([(s, c, n)], H, Hkv, DEV), SCALE)
        assert torch.equal(_bits(alone), _bits(out[row:row + n])), (s, c, n)
        row += n
    with pytest.raises(ValueError, match="plan is for"):  # a plan of another geometry
        ops.paged_prefill_attention_kv8(q, pool, t, ops.prefill_plan(chunks, H, Hkv * 2 if H > Hkv else 8, DEV), SCALE)


@pytest.mark.parametrize("ctx, n", [(20, 100), (3000, 9), (0, 70)])
def test_keys_that_are_not_finite_reach_only_the_rows_that_see_them(ctx, n):
    """NaN codes of later tokens of a chunk (and of what a recycled page holds past its end) leave a row as it is; a
    row that sees one gets NaN: all of it from K, that dim from V."""
    H, Hkv, L = 32, 4, ctx + n
    table, pages = _table([L], n)
    pool = ref.random_pool(pages, Hkv, n, DEV, v_spread=2.0)
    _poison_stale(pool, table, [L])
    t = torch.from_numpy(table).to(DEV)
    nan_v = {0: (ctx + n // 2, [3, 70, 127]), 1: (L - 1, [0]), 3: (ctx // 2, [64, 65])}  # head: (key, dims)
    nan_k = {2: ctx + n // 3}
    for h, (key, dims) in nan_v.items():
        pool[t[0, key // 16], h, ref.v_at(key % 16, torch.tensor(dims, device=DEV))] = 127 if h else 255
    for h, key in nan_k.items():
        pool[t[0, key // 16], h, ref.k_at(key % 16, torch.tensor([9], device=DEV))] = 255
    q = torch.randn((n, H, 128), generator=torch.Generator().manual_seed(n)).to(torch.bfloat16).to(DEV)
    out = ops.paged_prefill_attention_kv8(q, pool, _i32(table), ops.prefill_plan([(0, ctx, n)], H, Hkv, DEV), SCALE)
    last = ops.paged_decode_attention_kv8(q[-1:].contiguous(), pool, _i32(table), _i32([L]), L, SCALE)
    k, v = ref.read(pool, t[0])
    k, v = torch.nan_to_num(k[:, :L]), torch.nan_to_num(v[:, :L])
    seen = torch.arange(L, device=DEV)[None] <= ctx + torch.arange(n, device=DEV)[:, None]
    G = H // Hkv
    for h in range(Hkv):
        want, tol = ref.attend(q[:, h * G:(h + 1) * G], k[h], v[h], SCALE, seen)
        if h in nan_v:
            key, dims = nan_v[h]
            want[seen[:, key].nonzero()[:, 0][:, None], :, torch.tensor(dims, device=DEV)[None]] = float("nan")
        if h in nan_k:
            want[seen[:, nan_k[h]]] = float("nan")
        for got, rows in ((out, slice(0, n)), (last, slice(n - 1, n))):
            got, w, tl = got[:, h * G:(h + 1) * G].double(), want[rows], tol[rows]
            assert torch.equal(got.isnan(), w.isnan()), (h, ctx)
            assert bool(((got - w).abs() <= tl)[~w.isnan()].all()), (h, ctx)


def test_decode_of_more_sequences_than_a_launch_covers():
    B, H, Hkv = 4101, 8, 4
    rng = np.random.default_rng(1)
    lens = rng.integers(0, 40, B)
    lens[4096], lens[4095] = 700, 1100
    table, pages = _table(lens.tolist(), 1)
    table[:, 4:] = np.where(np.arange(4, table.shape[1])[None] < -(-lens[:, None] // 16), table[:, 4:], 0)
    pool = ref.random_pool(pages, Hkv, 1, DEV)
    q = torch.randn((B, H, 128), generator=torch.Generator().manual_seed(1)).to(torch.bfloat16).to(DEV)
    out = ops.paged_decode_attention_kv8(q, pool, _i32(table), _i32(lens), 16 * table.shape[1], SCALE)
    assert bool((out[torch.from_numpy(lens == 0).to(DEV)] == 0).all())
    some = [0, 1, 4094, 4095, 4096, 4097, 4100] + rng.integers(0, B, 60).tolist()
    some = [b for b in some if lens[b]]
    _check_decode(out[some], q[some], pool, torch.from_numpy(table[some]).to(DEV), [int(lens[b]) for b in some], "many")


def test_pools_past_4_gib():
    """Records whose offsets pass 32 bits: the same bits as in a small pool."""
    H, Hkv, lens, big = 32, 4, [70, 33], 260_000
    small_t, pages = _table(lens, 7, extra=0)
    n = sum(lens)
    far = np.random.default_rng(8).permutation(pages)
    ids = np.where(far % 2, big - 1 - far, far)  # half of the pages at either end
    pool, small = ops.kv8_pool(big, Hkv, DEV), ops.kv8_pool(pages, Hkv, DEV)
    assert pool.nbytes > 2 ** 32
    big_t = np.where(small_t < pages, ids[np.minimum(small_t, pages - 1)], 2 ** 31 - 1)
    g = torch.Generator().manual_seed(9)
    qkv = torch.randn((n, (H + 2 * Hkv) * 128), generator=g).to(torch.bfloat16).to(DEV)
    w, inv = torch.ones(128, dtype=torch.bfloat16, device=DEV), torch.rand(64, generator=g).to(DEV)
    outs = []
    for p, t in ((pool, big_t), (small, small_t)):
        t = _i32(t)
        st = ops.step_tables(_i32([0, 0]), _i32(lens), t, n)
        q = ops.qk_norm_rope_append_kv8(qkv, H, Hkv, w, w, 1e-6, inv, st.pos, st.slots, p)
        plan = ops.prefill_plan([(i, 0, m) for i, m in enumerate(lens)], H, Hkv, DEV)
        outs.append((_bits(q), _bits(ops.paged_prefill_attention_kv8(q, p, t, plan, SCALE)),
                     _bits(ops.paged_decode_attention_kv8(q[:2].contiguous(), p, t, st.lens, max(lens), SCALE))))
    assert all(torch.equal(a, b) for a, b in zip(*outs))
    assert torch.equal(pool[torch.from_numpy(ids).to(DEV)], small)
    src, dst = _i32([int(ids.max())]), _i32([big // 2])
    ops.kv8_copy_pages(pool, src, dst)
    assert torch.equal(pool[big // 2], pool[int(ids.max())]) and bool(pool[int(ids.max())].any())


def test_prompt_rows_after_262140_keys_of_16_heads():
    """The longest context: an expanded cache past 2 GiB, parts of the largest size."""
    H, ctx, n = 16, 262140, 4
    table, pages = _table([ctx + n], 5, extra=0)
    pool = ops.kv8_pool(pages, H, DEV)
    t = _i32(table)
    g = torch.Generator(device=DEV).manual_seed(5)
    for at in range(0, ctx + n, 65536):  # (rows of at most 65,535 a call)
        for lo, hi in ((at, at + 32768), (at + 32768, min(at + 65536, ctx + n))):
            k, v = (torch.randn((hi - lo, H, 128), generator=g, device=DEV).to(torch.bfloat16) for _ in range(2))
            st = ops.step_tables(_i32([lo]), _i32([hi - lo]), t, hi - lo)
            ops.kv8_append_paged(pool, k, v, st.slots)
    plan = ops.prefill_plan([(0, ctx, n)], H, H, DEV)
    assert ops.kv8_prefill_workspace_bytes(plan, H, H) > 2 ** 31
    q = torch.randn((n, H, 128), generator=g, device=DEV).to(torch.bfloat16)
    out = ops.paged_prefill_attention_kv8(q, pool, t, plan, SCALE)
    keep = torch.arange(ctx + n, device=DEV)[None] <= ctx + torch.arange(n, device=DEV)[:, None]
    for h in (0, 7, 15):
        k, v = ref.read(pool[:, h:h + 1].contiguous(), torch.from_numpy(table).to(DEV)[0])
        want, tol = ref.attend(q[:, h:h + 1], k[0], v[0], SCALE, keep)
        assert bool(((out[:, h:h + 1].double() - want).abs() <= tol).all()), h


def test_prompt_attention_replays_over_new_contents():
    """A captured chunk (expansion, key parts, merge) replayed over other rows, keys and page tables."""
    H, Hkv, chunks = 32, 4, [(0, 1500, 20), (1, 0, 70)]
    lens = [c + n for _, c, n in chunks]
    plan = ops.prefill_plan(chunks, H, Hkv, DEV)
    assert plan.kv8.slots > 0
    tables = [_table(lens, s, extra=0) for s in (1, 2, 3)]
    pools = [ref.random_pool(tables[0][1], Hkv, s, DEV) for s in (4, 5, 6)]
    g = torch.Generator().manual_seed(2)
    qs = [torch.randn((90, H, 128), generator=g).to(torch.bfloat16).to(DEV) for _ in range(3)]
    q, pool, t = qs[0].clone(), pools[0].clone(), _i32(tables[0][0])
    ops.paged_prefill_attention_kv8(q, pool, t, plan, SCALE)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = ops.paged_prefill_attention_kv8(q, pool, t, plan, SCALE)
    for i in (0, 1, 2, 0):
        q.copy_(qs[i])
        pool.copy_(pools[i])
        t.copy_(_i32(tables[i][0]))
        graph.replay()
        want = ops.paged_prefill_attention_kv8(qs[i], pools[i], _i32(tables[i][0]), plan, SCALE)
        assert torch.equal(_bits(out), _bits(want)), i
