"""Scores of given texts and beam search over an Engine's model and pool.

No counterpart in the reference, whose engine draws one continuation of a prompt and reports no probabilities.

A text's score comes from its prompt chunks' rows and the packed head (CausalLM.score): no [T, V] logits are made.

A search keeps its beams' books on the device: page tables, lengths, reference counts and a free list of pages that the pool
has lent it.  A step selects the continuations (token_logprobs, beam_select), lets the beams' sequences go on from their
parents' pages (pages_fork, kv_copy_pages_layers), takes the next pages (step_tables) and decodes.  The host knows every
row's position without reading anything back -- the beams of a prompt are equally long, and an ended one lets its pages go
and is decoded into a spare page -- so it waits for the device once in _CHECK steps, to see whether all have ended.
"""

from __future__ import annotations

import itertools
from dataclasses import dataclass

import numpy as np
import torch

from . import ops
from .kvpool import PoolExhausted, pages_for
from .model import make_step_state
from .ops import PAGE

_CHECK = 16  # steps between looks at whether every beam has ended
_ids = itertools.count()


@dataclass
class Beam:
    """One continuation of a prompt: its tokens (the end-of-sequence token included), the sum of their log-probabilities,
    and whether it ended on an end-of-sequence token."""

    tokens: list
    score: float
    finished: bool


def _make_room(eng, pages: int) -> None:
    """Evict stored prefixes until `pages` pages that no admitted request is owed are free; none where that many cannot
    come free (PoolExhausted)."""
    held = 0 if eng.store is None else eng.store.held_alone()
    most = eng.pool.free_pages + held - eng.outstanding
    if most < pages:
        raise PoolExhausted(f"{pages} pages needed, {most} free or held by stored prefixes alone")
    if eng.store is not None:
        eng.store.make_room(pages + eng.outstanding)


def _prompt(eng, tokens) -> list:
    tokens = [int(t) for t in tokens]
    if not tokens:
        raise ValueError("empty prompt")
    if min(tokens) < 0 or max(tokens) >= eng.lm.vocab:
        raise ValueError(f"prompt token ids must lie in [0, {eng.lm.vocab})")
    return tokens


def score(eng, tokens) -> list:
    """The log-probability of each token of a text but the first, given those before it."""
    tokens = _prompt(eng, tokens)
    n, step, sid, out = len(tokens) - 1, eng.prefill_chunk, ("score", next(_ids)), []
    if n == 0:
        return []
    _make_room(eng, pages_for(n))
    try:
        eng.pool.reserve(sid, n)
        for c in range(0, n, step):
            m = min(step, n - c)
            x = eng.forward_chunk(sid, tokens, c, m)
            nxt = ops.upload(np.asarray(tokens[c + 1:c + 1 + m], np.int32), eng.device)
            out.append(eng.lm.score(x, nxt).logprob)
    finally:
        eng.pool.release(sid)
    return torch.cat(out).tolist()


def beam_search(eng, prompts, beams: int, max_tokens: int, eos=None) -> list:
    """The `beams` best continuations of each prompt by the sum of their tokens' log-probabilities, the best first: a list
    of Beam a prompt (fewer where the model gives fewer)."""
    prompts = [_prompt(eng, p) for p in prompts]
    beams, max_tokens, lm, pool, dev = int(beams), int(max_tokens), eng.lm, eng.pool, eng.device
    if not 1 <= beams <= min(ops.BEAMS_MAX, lm.vocab):
        raise ValueError(f"beams must lie in [1, {min(ops.BEAMS_MAX, lm.vocab)}], got {beams}")
    if max_tokens < 1:
        raise ValueError("max_tokens must be >= 1")
    G, n = len(prompts), beams
    if G * n > eng.max_step_tokens:
        raise ValueError(f"{G} prompts of {n} beams pass a step's {eng.max_step_tokens} rows")
    if G == 0:
        return []
    eos = sorted({int(e) for e in (lm.eos_ids if eos is None else eos)})
    last = [len(p) + max_tokens - 1 for p in prompts]  # positions that a beam can come to hold
    # a beam's own pages: those past the prompt's full ones; a fork takes its copies before it gives pages back
    lent = 1 + sum(n * (pages_for(t) - len(p) // PAGE) + n for p, t in zip(prompts, last))
    _make_room(eng, lent + sum(pages_for(len(p)) for p in prompts))
    sids, pages = [("beams", next(_ids)) for _ in prompts], []
    try:
        h = []
        for sid, p in zip(sids, prompts):
            at, shared = eng.lookup(p)
            pool.open(sid, shared, at)
            while at < len(p):
                m = min(eng.prefill_chunk - at % eng.prefill_chunk, len(p) - at)
                pool.prepare_write(sid, at, m)
                x = eng.forward_chunk(sid, p, at, m)
                at += m
            pool.set_length(sid, at)
            h.append(x[-1:])
        pages = pool.alloc(lent)
        return _search(eng, prompts, sids, torch.cat(h), pages, n, max_tokens, eos, pages_for(max(last)))
    finally:
        pool.decref(pages)
        for sid in sids:
            pool.release(sid)


def _search(eng, prompts, sids, h, pages, n: int, max_tokens: int, eos: list, width: int) -> list:
    lm, pool, dev, i32 = eng.lm, eng.pool, eng.device, torch.int32
    G, lens_host = len(prompts), np.array([len(p) for p in prompts], np.int32)
    spare, free = pages[0], ops.upload(np.asarray(pages[1:], np.int32), dev)
    # the pool's hold on the prompts' pages stays: the beams' come on top, and no prompt page is written or given back
    table = pool.page_table(sids, width)
    counts = pool.refs.copy()
    counts[pages] = 0
    for sid in sids:
        counts[pool.pages[sid]] += 1
    refs, lens = ops.upload(counts, dev), ops.upload(lens_host, dev)
    at = torch.zeros(1, dtype=i32, device=dev)
    index = torch.arange(free.numel(), device=dev)
    ends = ops.upload(np.asarray(eos, np.int32), dev) if eos else None
    scores, done, rows = torch.zeros((G, 1), device=dev), None, 1
    parents, tokens, statuses, layers = [], [], [], pool.layers()
    for t in range(max_tokens):
        lp = ops.token_logprobs(lm.logits(h), top=n)
        b = ops.beam_select(scores, lp.top_logprobs.view(G, rows, n), lp.top_ids.view(G, rows, n), n, done, ends)
        scores, done, rows = b.scores, b.done, n
        parents.append(b.parents)
        tokens.append(b.tokens)
        if t + 1 == max_tokens or (t % _CHECK == _CHECK - 1 and bool(done.all())):
            break
        # (an ended beam, or one that is none, needs no pages any more)
        go = torch.where(done == 0, b.parents, -1).view(-1)
        f = ops.pages_fork(table, lens, go, refs, free, at)
        ops.kv_copy_pages_layers(layers, f.src, f.dst)
        on = go >= 0
        s = ops.step_tables(f.lens, on.to(i32), f.page_table, G * n, free, f.status[1:2])
        pos = np.repeat(lens_host + t, n)
        if (pos % PAGE == 0).any():  # pages taken from the list have one holder
            refs.index_add_(0, free, ((index >= f.status[1]) & (index < s.status[1])).to(i32))
        statuses += [f.status, s.status]
        table, lens, at = f.page_table, s.lens, s.status[1:2]
        st = make_step_state(lm.cfg, pos, torch.where(on[:, None], table, spare), pool.kv8)
        h = lm.model.decode_step(lm.embed_tokens(b.tokens.view(-1).clamp_min(0)), pool.pools, st)
    if statuses and bool(torch.stack(statuses)[:, 2].any()):
        raise PoolExhausted("a search's beams ran out of the pages lent to it")
    par, tok = (torch.stack(x).view(len(x), -1).tolist() for x in (parents, tokens))
    out, end, total = [], set(eos), scores.view(-1).tolist()
    for g in range(G):
        group = []
        for i in range(g * n, (g + 1) * n):
            if par[-1][i] < 0:
                continue
            seq, row = [], i
            for p, k in zip(reversed(par), reversed(tok)):
                if k[row] >= 0:
                    seq.append(k[row])
                row = p[row]
            seq.reverse()
            group.append(Beam(seq, total[i], bool(seq) and seq[-1] in end))
        out.append(group)
    return out
