"""The 8-bit cache as the model and the engine use it, on MI355X: the native layer calls against the op-by-op path (the
same bits), a mixed step's and a decode step's attention against 64 bits over what the cache holds, generations that
depend on their request alone, shared prefixes, and the registered operators against the library calls."""

from __future__ import annotations

import numpy as np
import pytest
import torch

from jitengine_amd import ops, torch_ops
from jitengine_amd.engine import Engine
from jitengine_amd.kvpool import KVPool
from jitengine_amd.model import MoEConfig, make_mixed_state, make_step_state, random_causal_lm
from tests import kv8_ref as ref

pytestmark = pytest.mark.gpu
DEV = "cuda"
CFG = MoEConfig(layers=2, experts=32)
VOCAB = 2048
SCALE = 128 ** -0.5


@pytest.fixture(scope="module")
def lm():
    return random_causal_lm(CFG, VOCAB, seed=11, device=DEV)


def _x(rows, seed):
    return torch.randn((rows, CFG.hidden), generator=torch.Generator().manual_seed(seed)).to(torch.bfloat16).to(DEV)


def _pools(seed, pages):
    return [ref.random_pool(pages, CFG.kv_heads, seed + i, DEV) for i in range(CFG.layers)]


def _tables(n, width, pages, seed):
    return np.random.default_rng(seed).permutation(pages)[:n * width].reshape(n, width).astype(np.int32)


def _check_rows(attn, q, pool, rows):
    """attn rows r against 64-bit attention over the first n keys of the given pages: rows [(r, pages, n)]."""
    G = CFG.heads // CFG.kv_heads
    for r, pages, n in rows:
        k, v = ref.read(pool, pages[:-(-n // 16)])
        for h in range(CFG.kv_heads):
            want, tol = ref.attend(q[r:r + 1, h * G:(h + 1) * G], k[h, :n], v[h, :n], SCALE)
            err = (attn[r:r + 1, h * G:(h + 1) * G].double() - want).abs()
            assert bool((err <= tol).all()), (r, n, h, float((err / tol).max()))


@pytest.mark.parametrize("pos", [[40], [0], [0, 15, 16, 517, 63], list(range(0, 280, 7))])
def test_decode_steps_native_and_op_by_op_agree(lm, pos):
    width = 36
    pages = len(pos) * width + 2
    table = torch.from_numpy(_tables(len(pos), width, pages, len(pos))).to(DEV)
    x, a = _x(len(pos), 3), _pools(5, pages)
    b = [p.clone() for p in a]
    st = make_step_state(CFG, pos, table, kv8=True)
    got = lm.model.decode_step(x, a, st)
    y, dbg = x, [{} for _ in lm.layers]
    for layer, pool, d in zip(lm.layers, b, dbg):
        y = layer.step(y, pool, st, debug=d)
    assert torch.equal(got, y) and all(torch.equal(p, q) for p, q in zip(a, b))
    _check_rows(dbg[1]["attn"], dbg[1]["q"], b[1], [(r, table[r].tolist(), p + 1) for r, p in enumerate(pos)])


@pytest.mark.parametrize("chunks, dec", [
    ([(0, 0, 1)], []), ([(0, 33, 40), (1, 0, 17)], [5, 100]), ([(1, 100, 300)], [0]), ([], [3, 31, 200]),
    ([(0, 16, 16), (0, 32, 9)], []),
])
def test_mixed_steps_native_and_op_by_op_agree(lm, chunks, dec):
    width, layer = 26, lm.layers[0]
    S, D = 2, len(dec)
    pages = (S + D) * width + 1
    tab = _tables(S + D, width, pages, 9 + D)
    ms = make_mixed_state(CFG, chunks, tab[:S], dec, tab[S:], DEV, kv8=True)
    T = sum(n for *_, n in chunks) + D
    assert ms.P == T - D and ms.kv8.pos.tolist() == [c + i for _, c, n in chunks for i in range(n)] + dec
    x, a = _x(T, 4), _pools(7, pages)[0]
    b, dbg = a.clone(), {}
    got = layer.mixed(x, a, ms)
    assert torch.equal(got, layer.mixed(x, b, ms, debug=dbg)) and torch.equal(a, b)
    rows, r = [], 0
    for s, c, n in chunks:
        rows += [(r + i, tab[s].tolist(), c + i + 1) for i in (0, n // 2, n - 1)]
        r += n
    rows += [(r + i, tab[S + i].tolist(), p + 1) for i, p in enumerate(dec)]
    _check_rows(dbg["attn"], dbg["q"], b, rows)


def test_steps_refuse_rows_and_pools_of_another_kind(lm):
    table = torch.arange(8, dtype=torch.int32, device=DEV).view(2, 4)
    st8, st = (make_step_state(CFG, [3, 9], table, kv8) for kv8 in (True, False))
    p8, p = KVPool(2, 8, CFG.kv_heads, DEV, kv8=True).pools, KVPool(2, 8, CFG.kv_heads, DEV).pools
    for pools, state, x in ((p8, st, _x(2, 1)), (p, st8, _x(2, 1)), (p8, st8, _x(3, 1)), (p8, st8, _x(1, 1)),
                            (p8, st8, _x(2, 1).float()), (KVPool(2, 8, 8, DEV, kv8=True).pools, st8, _x(2, 1)),
                            ([p8[0], p[1]], st8, _x(2, 1))):
        with pytest.raises(ValueError):
            lm.model.decode_step(x, pools, state)
    ms = make_mixed_state(CFG, [(0, 0, 3)], table[:1].cpu().numpy(), [2], table[1:].cpu().numpy(), DEV, kv8=True)
    for pool, x in ((p[0], _x(4, 1)), (p8[0], _x(5, 1)), (p8[0], _x(3, 1))):
        with pytest.raises(ValueError):
            lm.layers[0].mixed(x, pool, ms)


def _prompts(seed, lens):
    rng = np.random.default_rng(seed)
    return [rng.integers(0, VOCAB, n).tolist() for n in lens]


def _solo(lm, prompt, max_tokens, **kw):
    e = Engine(lm, 64, prefill_chunk=16, max_step_tokens=48, prefix_store=False, pipeline=False, kv8=True)
    r = e.submit(prompt, max_tokens, eos=(), **kw)
    e.run()
    return r.tokens


@pytest.mark.parametrize("pipeline", [False, True])
def test_engine_batched_equals_solo(lm, pipeline):
    prompts = _prompts(1, [5, 17, 33, 40, 9])
    kws = [{}, dict(temperature=0.8, top_p=0.9, top_k=40, seed=5), {}, {}, dict(temperature=1.2, seed=6)]
    e = Engine(lm, 128, prefill_chunk=16, max_step_tokens=48, page_seed=7, selfcheck=True, kv8=True, pipeline=pipeline)
    reqs = [e.submit(p, 9, eos=(), **kw) for p, kw in zip(prompts[:2], kws)]
    e.step()
    e.step()
    reqs += [e.submit(p, 9, eos=(), **kw) for p, kw in zip(prompts[2:], kws[2:])]
    e.run()
    for r, p, kw in zip(reqs, prompts, kws):
        assert r.finish_reason == "length" and r.tokens == _solo(lm, p, 9, **kw), r.rid


def test_engine_prefix_sharing_is_exact(lm):
    base, = _prompts(2, [40])
    ext = _prompts(3, [10, 7])
    e = Engine(lm, 128, prefill_chunk=24, max_step_tokens=48, kv8=True)
    a = e.submit(base, 4, eos=())
    e.run()
    stored = list(e.store.entries[tuple(base)])
    before = [p[stored].clone() for p in e.pool.pools]
    b = e.submit(base + ext[0], 5, eos=())
    c = e.submit(base + ext[1], 5, eos=())
    e.run()
    assert b.cached == 24 and c.cached == 24 and e.pool.copies >= 2
    assert all(torch.equal(p[stored], x) for p, x in zip(e.pool.pools, before))  # never written
    for r, p in ((a, base), (b, base + ext[0]), (c, base + ext[1])):
        e1 = Engine(lm, 64, prefill_chunk=24, max_step_tokens=48, prefix_store=False, kv8=True)
        want = e1.submit(p, len(r.tokens), eos=())
        e1.run()
        assert r.tokens == want.tokens


def test_registered_operators_equal_the_library_calls():
    J = torch.ops.jitengine
    H, Hkv, S, W = 32, 4, 3, 40
    g = torch.Generator().manual_seed(2)

    def bf(*shape):
        return torch.randn(shape, generator=g).to(torch.bfloat16).to(DEV)

    def i32(a):
        return torch.tensor(a, dtype=torch.int32, device=DEV)

    new, rows = [1, 20, 600], 621
    a, b = (ref.random_pool(S * W, Hkv, 4, DEV) for _ in range(2))
    ta, tb = (i32(np.full((S, W), -1)) for _ in range(2))
    free = i32(np.random.default_rng(5).permutation(S * W))
    args = (i32([0, 0, 0]), i32(new))
    t = ops.step_tables(*args, ta, rows, free)
    got = J.step_tables(*args, tb, rows, free, None)
    want = (t.row_start, t.row_seq, t.pos, t.slots, t.lens, t.status)
    assert all(torch.equal(x, y) for x, y in zip(got, want)) and torch.equal(ta, tb)
    qkv, qn, kn, inv = bf(rows, (H + 2 * Hkv) * 128), bf(128), bf(128), torch.rand(64, generator=g).to(DEV)
    append = (qkv, H, Hkv, qn, kn, 1e-6, inv, t.pos, t.slots)
    q = ops.qk_norm_rope_append_kv8(*append, a)
    assert torch.equal(J.qk_norm_rope_append_kv8(*append, b), q) and torch.equal(a, b)
    plan = ops.prefill_plan([(i, 0, n) for i, n in enumerate(new)], H, Hkv, DEV)
    pws = torch.empty(ops.kv8_prefill_workspace_bytes(plan, H, Hkv), dtype=torch.uint8, device=DEV)
    pargs = (q, a, ta, *torch_ops.kv8_prefill_plan_args(plan), SCALE, pws)
    assert torch.equal(J.paged_prefill_attention_kv8(*pargs), ops.paged_prefill_attention_kv8(q, a, ta, plan, SCALE))
    dws = torch.empty(ops.kv8_decode_workspace_bytes(S, H, 600), dtype=torch.uint8, device=DEV)
    tc = torch.where(ta < 0, torch.zeros_like(ta), ta)
    dargs = (q[:S].contiguous(), a, tc, t.lens, 600, SCALE)
    assert torch.equal(J.paged_decode_attention_kv8(*dargs, dws), ops.paged_decode_attention_kv8(*dargs))
    k, v = bf(rows, Hkv, 128), bf(rows, Hkv, 128)
    ops.kv8_append_paged(a, k, v, t.slots)
    J.kv8_append_paged(b, k, v, t.slots)
    assert torch.equal(a, b)
    src, dst = t.slots[-17:-16] // 16, free[-1:]
    ops.kv8_copy_pages(a, src, dst)
    J.kv8_copy_pages(b, src, dst)
    assert torch.equal(a, b) and torch.equal(a[int(dst)], a[int(src)])
    cases = [(J.step_tables, (*args, tb, rows, free, None)), (J.qk_norm_rope_append_kv8, (*append, b)),
             (J.paged_prefill_attention_kv8, pargs), (J.paged_decode_attention_kv8, (*dargs, dws)),
             (J.kv8_append_paged, (b, k, v, t.slots)), (J.kv8_copy_pages, (b, src, dst))]
    assert {op._qualified_op_name.split("::")[1] for op, _ in cases} == set(torch_ops.OPS_KV8)
    for op, op_args in cases:
        torch.library.opcheck(op, op_args)


def test_the_registered_step_tables_is_one_launch():
    """Into outputs of their own: no copies after it."""
    ctx, new, table = (torch.tensor(x, dtype=torch.int32, device=DEV) for x in ([3, 40], [5, 1], [[0, 1, 2], [3, 4, 5]]))
    J = torch.ops.jitengine
    got = J.step_tables(ctx, new, table, 6, None, None)
    with torch.profiler.profile(activities=[torch.profiler.ProfilerActivity.CUDA]) as prof:
        got = J.step_tables(ctx, new, table, 6, None, None)
        torch.cuda.synchronize()
    names = [e.key for e in prof.key_averages() for _ in range(e.count) if e.self_device_time_total > 0]
    assert len(names) == 1 and "step_tables_kernel" in names[0], names
    assert len({t.untyped_storage().data_ptr() for t in got}) == 6
    assert got[3].tolist() == [3, 4, 5, 6, 7, 16 * 5 + 8] and got[4].tolist() == [8, 41]
