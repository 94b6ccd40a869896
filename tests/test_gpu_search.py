"""Scores, searches and per-token log-probabilities of an engine on the GPU, and the operators' torch forms.

A search is compared with a plain one, in 64 bits on the host, whose every step decodes each continuation through pages of
its own; the rows of a decode step do not depend on the batch, so both see the same logits."""

from __future__ import annotations

import numpy as np
import pytest
import torch

from jitengine_amd import ops, torch_ops
from jitengine_amd.engine import Engine
from jitengine_amd.model import MoEConfig, make_step_state, random_causal_lm
from tests.test_gpu_scoring import U, _head_ref, _i32
from jitengine_amd.quant import random_quantized

pytestmark = pytest.mark.gpu
DEV = "cuda"
VOCAB = 2048


@pytest.fixture(scope="module")
def lm():
    return random_causal_lm(MoEConfig(layers=2, experts=32), VOCAB, seed=21, device=DEV, std=0.04)


def _prompt(n, seed):
    return np.random.default_rng(seed).integers(0, VOCAB, n).tolist()


def _engine(lm, pages=256, chunk=32, **kw):
    return Engine(lm, pages, prefill_chunk=chunk, max_step_tokens=64, device=DEV, page_seed=5, **kw)


def _plain(lm, prompt, beams, max_tokens, eos, kv8):
    """The search with a sequence of the pool for each continuation, scores in 64 bits."""
    eng = _engine(lm, 512, prefix_store=False, kv8=kv8)
    pool, at = eng.pool, 0
    pool.reserve("p", len(prompt))
    while at < len(prompt):
        m = min(32, len(prompt) - at)
        h = eng.forward_chunk("p", prompt, at, m)[-1:]
        at += m
    live = [([], 0.0, False, "p", h)]
    for t in range(max_tokens):
        cands = []
        for i, (toks, s, ended, sid, h) in enumerate(live):
            if ended:
                cands.append((s, i, 0, None))
                continue
            lp = torch.log_softmax(lm.logits(h)[0].double().cpu(), -1)
            best = sorted(range(VOCAB), key=lambda v: (-float(lp[v]), v))[:beams]
            cands += [(s + float(lp[v]), i, j, v) for j, v in enumerate(best)]
        cands.sort(key=lambda c: (-c[0], c[1], c[2]))
        nxt = []
        for k, (s, i, _, v) in enumerate(cands[:beams]):
            toks, _, _, sid, _ = live[i]
            if v is None:
                nxt.append((toks, s, True, None, None))
                continue
            new, pos = (t, k), len(prompt) + t
            pool.open(new, pool.pages[sid], pos)
            pool.prepare_write(new, pos, 1)
            st = make_step_state(lm.cfg, np.array([pos], np.int32), pool.page_table([new]), kv8)
            h = lm.model.decode_step(lm.embed_tokens(_i32([v])), pool.pools, st)
            nxt.append((toks + [v], s, v in eos, new, h))
        live = nxt
    return [(toks, s, ended) for toks, s, ended, _, _ in live]


def _same(got, want):
    assert [b.tokens for b in got] == [w[0] for w in want] and [b.finished for b in got] == [w[2] for w in want]
    for b, w in zip(got, want):
        # a step adds a log-probability (off by 100 half steps of its row's sum, rounded) and rounds the score
        steps = len(w[0])
        assert abs(b.score - w[1]) <= steps * (100 * U + 2 * U * abs(w[1]))


@pytest.mark.parametrize("kv8", [False, True])
@pytest.mark.parametrize("length,beams,max_tokens", [(1, 1, 3), (16, 4, 20), (37, 3, 18), (47, 8, 2), (70, 5, 1)])
def test_beam_search_is_the_plain_one(lm, length, beams, max_tokens, kv8):
    prompt = _prompt(length, length)
    eng = _engine(lm, kv8=kv8)
    want = _plain(lm, prompt, beams, max_tokens, (), kv8)
    _same(eng.beam_search([prompt], beams, max_tokens, eos=())[0], want)
    assert not eng.pool.refs.any() and eng.pool.free_pages == 256 and not eng.pool.pages


def test_beams_end_and_go_on(lm):
    """Continuations that end are kept as they are beside the others; a search whose every beam has ended stops."""
    prompt, eng = _prompt(20, 3), _engine(lm)
    free = eng.beam_search([prompt], 4, 24, eos=())[0]
    eos = sorted({b.tokens[i] for b, i in zip(free, (2, 5, 9, 13))})
    got = eng.beam_search([prompt], 4, 24, eos=eos)[0]
    assert any(b.finished for b in got)
    _same(got, _plain(lm, prompt, 4, 24, set(eos), False))
    got = eng.beam_search([prompt], 3, 40, eos=range(VOCAB))[0]  # whatever comes ends
    assert all(b.finished and len(b.tokens) == 1 for b in got)
    assert eng.pool.free_pages == 256


def test_searches_of_several_prompts_beside_requests(lm):
    """Prompts of different lengths searched together give what each gives alone, restored prefixes and running requests
    included, and leave both as they were."""
    prompts = [_prompt(n, n) for n in (5, 64, 33)]
    want = [_engine(lm).beam_search([p], 4, 12)[0] for p in prompts]
    alone = _engine(lm)
    ra = alone.submit(prompts[1] + [7], 10, eos=())
    alone.run()
    eng = _engine(lm)
    first = eng.submit(prompts[1] + [9], 2, eos=())
    eng.run()  # (leaves its prompt in the store)
    r = eng.submit(prompts[1] + [7], 10, eos=())
    for _ in range(4):
        eng.step()
    free, refs = eng.pool.free_pages, eng.pool.refs.copy()
    got = eng.beam_search(prompts, 4, 12)
    for g, w in zip(got, want):
        assert [(b.tokens, b.score, b.finished) for b in g] == [(b.tokens, b.score, b.finished) for b in w]
    assert eng.pool.free_pages == free and np.array_equal(eng.pool.refs, refs)
    eng.run()
    assert first.state == r.state == "done" and r.tokens == ra.tokens


def test_a_search_of_rows_without_numbers_ends_empty(lm):
    class Dead:
        cfg, layers, vocab, eos_ids, model = lm.cfg, lm.layers, lm.vocab, (), lm.model
        embed_tokens = staticmethod(lm.embed_tokens)
        final_norm = lm.final_norm

        @staticmethod
        def logits(h):
            return torch.full((h.shape[0], VOCAB), float("nan"), dtype=torch.bfloat16, device=DEV)

    eng = _engine(Dead)
    assert eng.beam_search([_prompt(30, 1)], 4, 6) == [[]]
    assert eng.pool.free_pages == 256
    untouched = np.setdiff1d(np.arange(256), eng.pool._free[-64:])
    assert all(not p[torch.from_numpy(untouched).to(DEV)].any() for p in eng.pool.pools)


@pytest.mark.parametrize("kv8", [False, True])
@pytest.mark.parametrize("n", [2, 17, 33, 65, 130])
def test_score_of_a_text(lm, n, kv8):
    tokens = _prompt(n, 50 + n)
    eng = _engine(lm, kv8=kv8)
    got = eng.score(tokens)
    assert len(got) == n - 1 and eng.pool.free_pages == 256
    ref = _engine(lm, kv8=kv8)
    ref.pool.reserve("p", n)
    lin = random_quantized((VOCAB, lm.cfg.hidden), 21 * 10 + 9, 0.04, DEV)  # (the model's head before its packing)
    at = 0
    while at < n - 1:
        m = min(32, n - 1 - at)
        x = ops.rmsnorm(ref.forward_chunk("p", tokens, at, m), lm.final_norm, lm.cfg.eps)
        lp, _, _, bound = _head_ref(x, lin, _i32(tokens[at + 1:at + 1 + m]))
        diff = (torch.tensor(got[at:at + m], device=DEV).double() - lp).abs()
        assert torch.all(diff <= 2 * bound + (VOCAB / 256 + 128) * U + U * lp.abs())
        at += m


@pytest.mark.parametrize("temperature", [0.0, 0.9])
@pytest.mark.parametrize("pipeline", [False, True])
@pytest.mark.parametrize("top", [0, 1, 20])
def test_log_probabilities_of_generated_tokens(lm, top, pipeline, temperature):
    """The tokens are those of a request that asks for none; each one's numbers are those of the logits it was drawn from."""
    prompt, kw = _prompt(40, 9), dict(eos=(), temperature=temperature, seed=3)
    plain = _engine(lm, pipeline=pipeline)
    want = plain.submit(prompt, 9, **kw)
    plain.run()
    seen = []

    class Seen:
        cfg, layers, vocab, eos_ids, model = lm.cfg, lm.layers, lm.vocab, (), lm.model
        embed_tokens, greedy = staticmethod(lm.embed_tokens), staticmethod(lm.greedy)
        final_norm = lm.final_norm

        @staticmethod
        def logits(h):
            seen.append(lm.logits(h))
            return seen[-1]

    eng = _engine(Seen, pipeline=pipeline)
    r = eng.submit(prompt, 9, logprobs=top, **kw)
    eng.run()
    assert r.tokens == want.tokens and len(r.logprobs) == len(r.tokens) == len(seen) and not want.logprobs
    for c, t, x in zip(r.logprobs, r.tokens, seen):
        x = x[0].double().cpu()
        lp = torch.log_softmax(x, -1)
        order = sorted(range(VOCAB), key=lambda v: (-float(x[v]), v))
        assert abs(c.logprob - float(lp[t])) <= 100 * U + U * abs(float(lp[t])) and c.rank == order.index(t)
        assert [v for v, _ in c.top] == order[:top]
        for v, p in c.top:
            assert abs(p - float(lp[v])) <= 100 * U + U * abs(float(lp[v]))


def test_log_probabilities_beside_requests_without(lm):
    """Requests of one step that ask for different numbers of alternatives, or for none; one that ends on a token."""
    prompts = [_prompt(n, n) for n in (12, 20, 31)]
    alone = []
    for p, top in zip(prompts, (None, 2, 5)):
        eng = _engine(lm)
        alone.append(eng.submit(p, 8, eos=(), logprobs=top))
        eng.run()
    stop = alone[1].tokens[3]
    eng = _engine(lm)
    rs = [eng.submit(p, 8, eos=(stop,) if i == 1 else (), logprobs=top) for i, (p, top) in enumerate(zip(prompts, (None, 2, 5)))]
    eng.run()
    n = alone[1].tokens.index(stop) + 1
    assert rs[0].tokens == alone[0].tokens and rs[1].tokens == alone[1].tokens[:n] and rs[2].tokens == alone[2].tokens
    assert not rs[0].logprobs
    for r, a, top in ((rs[1], alone[1], 2), (rs[2], alone[2], 5)):
        assert len(r.logprobs) == len(r.tokens) and all(len(c.top) == top for c in r.logprobs)
        for c, d in zip(r.logprobs, a.logprobs):  # (the slices of a row depend on the batch: sums in another order)
            assert c.rank == d.rank and [v for v, _ in c.top] == [v for v, _ in d.top]
            assert abs(c.logprob - d.logprob) <= 200 * U + 2 * U * abs(d.logprob)


@pytest.mark.parametrize("kv8", [False, True])
def test_a_pool_copies_pages_in_every_layer(lm, kv8):
    eng = _engine(lm, 32, kv8=kv8)
    g = torch.Generator(device=DEV).manual_seed(4)
    for p in eng.pool.pools:
        p.copy_(torch.randint(0, 100, p.shape, generator=g, device=DEV).to(p.dtype))
    want = [p.clone() for p in eng.pool.pools]
    for w in want:
        (ops.kv8_copy_pages if kv8 else ops.kv_copy_pages)(w, _i32([3, 0, 3]), _i32([7, 30, 31]))
    eng.pool.copy_pages([3, 0, 3], [7, 30, 31])
    assert all(torch.equal(a, b) for a, b in zip(eng.pool.pools, want))
    eng.pool.pools = [p.clone() for p in eng.pool.pools]  # pools that took the place of others
    eng.pool.copy_pages([7], [9])
    assert all(torch.equal(p[7], p[9]) and not torch.equal(w[7], w[9]) for p, w in zip(eng.pool.pools, want))


def test_operators_as_torch_ops():
    J, g = torch.ops.jitengine, torch.Generator(device=DEV).manual_seed(8)
    x = torch.randn((3, 700), generator=g, device=DEV)
    tok = _i32([[5, 699], [0, -1], [33, 34]])
    a, b = J.token_logprobs(x, tok, 4), ops.token_logprobs(x, tok, 4)
    assert all(torch.equal(s, t) for s, t in zip(a, (b.logprob, b.rank, b.entropy, b.top_ids, b.top_logprobs)))
    lin = ops.prepack(random_quantized((512, 256), 1, device=DEV))
    h = torch.randn((20, 256), generator=g, device=DEV).to(torch.bfloat16)
    ht = _i32(np.arange(20))
    r = ops.head_logprobs(h, lin, ht)
    assert torch.equal(J.head_logprobs(h, lin.data, 512, 256, ht), torch.stack((r.logprob, r.entropy, r.lse)))
    sel = (b.logprob[:, :1].t().contiguous(), b.top_logprobs[None], b.top_ids[None], 5, None, _i32([7]))
    c, d = J.beam_select(*sel), ops.beam_select(*sel)
    assert all(torch.equal(s, t) for s, t in zip(c, (d.parents, d.tokens, d.scores, d.done)))
    fork = lambda: (_i32([[1, 2], [3, 0]]), _i32([20, 16]), _i32([0, 0, 1]), _i32([0, 1, 1, 1, 0, 0]), _i32([9, 4, 5, 0]), _i32([1]))
    fa, fb = fork(), fork()
    e, f = J.pages_fork(*fa), ops.pages_fork(*fb)
    assert all(torch.equal(s, t) for s, t in zip(e, (f.page_table, f.lens, f.src, f.dst, f.status)))
    assert all(torch.equal(s, t) for s, t in zip(fa, fb))
    pools = [torch.randn((6, 2, 2, 2048), generator=g, device=DEV).to(torch.bfloat16) for _ in range(3)]
    J.kv_copy_pages_layers(pools, _i32([1]), _i32([4]))
    assert all(torch.equal(p[1], p[4]) for p in pools)
    cases = [(J.token_logprobs, (x, tok, 4)), (J.token_logprobs, (x, tok, 0)), (J.head_logprobs, (h, lin.data, 512, 256, ht)),
             (J.beam_select, sel), (J.pages_fork, fork()), (J.kv_copy_pages_layers, (pools, _i32([1]), _i32([4])))]
    assert {op._qualified_op_name.split("::")[1] for op, _ in cases} == set(torch_ops.OPS_SCORING)
    for op, args in cases:
        torch.library.opcheck(op, args)
