"""Scoring, parallel continuations and beam search over a paged cache as calls that can be timed and compared: each operator
in its plain form (elementary torch operations, 32 bits) and as a program calls it of this framework.

Kinds of case:

  logprobs  of rows of logits: the log-probability and rank of a given token, the entropy, and the `top` most likely
            tokens with theirs (`ops.token_logprobs`);
  head      the log-probability of a given token, the entropy and the log of the sum of exponentials, from hidden rows
            and the 4-bit head matrix, without the logits in memory (`ops.head_logprobs`);
  beams     the best continuations of each group's beams from their alternatives (`ops.beam_select`);
  fork      the page tables, reference counts and free list after sequences were continued by others, with the list of
            pages to copy (`ops.pages_fork`);
  copy      cache pages copied in every layer (`ops.kv_copy_pages_layers`).

Order among equal values: the lowest index (token, candidate, page) first.

The head's 4-bit matrix [V, K] has groups of 64 along K with a bf16 scale s and bias b: w = s q + b, q in 0 .. 15.  For
every 16 rows the packed bytes hold K / 128 nibble tiles of 1,024 bytes, then K / 128 scale tiles of 128 bytes.  Lane 16 g
+ r of a nibble tile has 16 bytes of row r: the words 2 g and 2 g + 1 of the tile's first group of 64, then those of its
second; a word is 8 values, those of even index in its low half and those of odd index in its high half, 4 bits each.  A
scale tile has for each row the two groups' scales, then their biases.

A cache page holds 16 tokens.  A sequence of n tokens holds the first ceil(n / 16) pages of its table's row.
"""

from __future__ import annotations

import math
import random

import numpy as np
import torch

own = False

DEV = "cuda"
PAGE, PART = 16, 16 * 128


# ----------------------------------------------------------------------------- the cases
def listed() -> list:
    return [
        # one user's step with the usual handful of alternatives: the smallest call, latency alone
        {"name": "logprobs_1", "kind": "logprobs", "rows": 1, "vocab": 151936, "top": 5, "mask": 0.0},
        # a serving batch that asks for the most alternatives, under a grammar that rules most tokens out
        {"name": "logprobs_32_masked", "kind": "logprobs", "rows": 32, "vocab": 248320, "top": 20, "mask": 0.9},
        # the logits of a prompt chunk, scored with alternatives
        {"name": "logprobs_2048", "kind": "logprobs", "rows": 2048, "vocab": 151936, "top": 5, "mask": 0.0},
        # one row against the whole head: bound by the head's bytes
        {"name": "head_1", "kind": "head", "rows": 1, "hidden": 2048, "vocab": 151936},
        # the rest of a prompt past its last full chunk, odd in length
        {"name": "head_77", "kind": "head", "rows": 77, "hidden": 2048, "vocab": 151936},
        # four prompt chunks of 512 rows scored at once: bound by the matrix cores
        {"name": "head_2048", "kind": "head", "rows": 2048, "hidden": 2048, "vocab": 248320},
        # one request's four beams
        {"name": "beams_1x4", "kind": "beams", "groups": 1, "beams": 4, "alts": 8, "width": 4},
        # a batch of wide searches
        {"name": "beams_64x16", "kind": "beams", "groups": 64, "beams": 16, "alts": 32, "width": 16},
        # one request's eight beams over a prompt of some thousand tokens
        {"name": "fork_8", "kind": "fork", "groups": 1, "beams": 8, "prompt": 4096, "fresh": 256, "pages": 4096},
        # 64 requests of eight beams each
        {"name": "fork_512", "kind": "fork", "groups": 64, "beams": 8, "prompt": 8192, "fresh": 512, "pages": 65536},
        # the last pages of seven new continuations, in every layer
        {"name": "copy_7", "kind": "copy", "layers": 48, "kv_heads": 4, "pages": 256, "moved": 7},
        # a third of a pool moved together after its sequences have ended
        {"name": "copy_256", "kind": "copy", "layers": 48, "kv_heads": 4, "pages": 768, "moved": 256},
    ]


def _log(rng: random.Random, lo: int, hi: int) -> int:
    return max(lo, min(hi, round(math.exp(rng.uniform(math.log(lo), math.log(hi + 1))))))


def draw(rng: random.Random) -> dict:
    """A case of the ranges the listed ones stand for."""
    kind = rng.choice(["logprobs", "logprobs", "head", "head", "head", "beams", "fork", "copy"])
    if kind == "logprobs":
        return {"kind": kind, "rows": _log(rng, 1, 2048), "vocab": rng.choice([151936, 151936, 248320, _log(rng, 64, 200000)]),
                "top": rng.choice([0, 1, 2, 5, 8, 20, 32]), "mask": rng.choice([0.0, 0.0, 0.5, 0.99])}
    if kind == "head":
        return {"kind": kind, "rows": _log(rng, 1, 2048), "hidden": 128 * _log(rng, 1, 16),
                "vocab": rng.choice([151936, 248320, 16 * _log(rng, 8, 10000)])}
    if kind == "beams":
        beams = rng.randint(1, 16)
        alts = rng.randint(1, 32)
        return {"kind": kind, "groups": _log(rng, 1, 64), "beams": beams, "alts": alts, "width": rng.randint(1, 16)}
    if kind == "fork":
        groups, beams = _log(rng, 1, 64), rng.randint(1, 8)
        return {"kind": kind, "groups": groups, "beams": beams, "prompt": _log(rng, 1, 8192), "fresh": _log(rng, 1, 512),
                "pages": 65536}
    pages = _log(rng, 16, 768)
    return {"kind": kind, "layers": rng.choice([1, 12, 24, 48]), "kv_heads": rng.choice([1, 2, 4, 8]) if pages <= 384 else 4,
            "pages": pages, "moved": _log(rng, 1, pages // 3)}


# ----------------------------------------------------------------------------- inputs
def _gen(seed: int) -> torch.Generator:
    g = torch.Generator(device=DEV)
    g.manual_seed(int(seed))
    return g


def _dev(a, dtype=np.int32) -> torch.Tensor:
    return torch.from_numpy(np.ascontiguousarray(np.asarray(a).astype(dtype))).to(DEV)


def _logits(g, case: dict):
    """Rows of a peaked, long-tailed distribution, and a token drawn from each."""
    n, v = case["rows"], case["vocab"]
    x = torch.randn((n, v), generator=g, device=DEV)
    x = 2.0 * x + 0.25 * x * x.abs()
    if case["mask"] > 0:
        out = torch.rand((n, v), generator=g, device=DEV) < case["mask"]
        out[:, 7] = False
        x.masked_fill_(out, -math.inf)
        del out
    x = x.to(torch.bfloat16)
    noise = torch.empty((n, v), device=DEV).exponential_(generator=g)
    tok = (x.float() - torch.log(noise)).argmax(-1).to(torch.int32)
    return x, tok


def _head(g, v: int, k: int):
    """The head's packed bytes: words of random 4-bit values, scales and biases of rows of N(0, 0.02) weights."""
    blocks, gp = v // 16, k // 128
    nib = torch.randint(-2 ** 31, 2 ** 31, (blocks, gp * 256), generator=g, device=DEV, dtype=torch.int64).to(torch.int32)
    s = 0.005 * (0.75 + 0.5 * torch.rand((blocks, gp, 16, 2), generator=g, device=DEV))
    b = s * (-7.5 + 0.5 * torch.randn(s.shape, generator=g, device=DEV))
    sc = torch.cat([s, b], -1).to(torch.bfloat16).contiguous().view(torch.int32).view(blocks, gp * 32)
    return torch.cat([nib, sc], 1).contiguous().view(torch.uint8).reshape(-1)


def _fork_tables(rng, case: dict) -> dict:
    """Groups of beams: the full pages of a group's prompt are shared by its beams, the pages after them are each beam's
    own; some beams end, others are continued several times."""
    gr, n, w = case["groups"], case["beams"], case["pages"]
    s = gr * n
    prompt = np.maximum(1, rng.integers(case["prompt"] // 2, case["prompt"] + 1, gr)) if case["prompt"] > 1 else np.ones(gr, np.int64)
    fresh = rng.integers(0, case["fresh"] + 1, gr)
    lens = np.repeat(prompt + fresh, n)
    shared = np.repeat(prompt // PAGE, n)                       # full pages of the prompt
    held = -(-lens // PAGE)
    width = -(-(case["prompt"] + case["fresh"]) // PAGE) + 2
    perm = rng.permutation(w)
    group = np.repeat(np.arange(gr), n)
    at = np.concatenate([[0], np.cumsum(prompt // PAGE)])       # where each group's shared pages stand in perm
    mine = np.concatenate([[0], np.cumsum(held - shared)]) + at[-1]
    j = np.arange(width)[None]
    idx = np.where(j < shared[:, None], at[group][:, None] + j, mine[:-1][:, None] + j - shared[:, None])
    table = np.where(j < held[:, None], perm[np.clip(idx, 0, w - 1)], 0)
    used = int(mine[-1])
    if used + s > w:
        raise ValueError(f"{used} pages and {s} copies do not fit {w}")
    refs = np.bincount(table[j < held[:, None]], minlength=w)
    # the free list stands behind the pages taken from it
    parents = group * n + rng.integers(0, n, s)
    parents[rng.random(s) < 0.05] = -1
    return {"table": table, "lens": lens, "parents": parents, "refs": refs, "free": perm, "at": used}


def prepare(case: dict, seed: int) -> dict:
    g = _gen(seed)
    rng = np.random.default_rng([seed, 7])
    kind = case["kind"]
    if kind == "logprobs":
        x, tok = _logits(g, case)
        return {"case": case, "logits": x, "tokens": tok}
    if kind == "head":
        n, v, k = case["rows"], case["vocab"], case["hidden"]
        x = torch.randn((n, k), generator=g, device=DEV) * (1.0 + 0.3 * torch.randn(k, generator=g, device=DEV))
        return {"case": case, "x": x.to(torch.bfloat16), "head": _head(g, v, k), "tokens": _dev(rng.integers(0, v, n))}
    if kind == "beams":
        gr, n, m = case["groups"], case["beams"], case["alts"]
        lp = -torch.empty((gr, n, m), device=DEV).exponential_(0.4, generator=g).sort(-1).values
        ids = torch.randint(0, 151936, (gr, n, m), generator=g, device=DEV).to(torch.int32)
        done = torch.rand((gr, n), generator=g, device=DEV) < 0.15
        return {"case": case, "scores": -40.0 * torch.rand((gr, n), generator=g, device=DEV), "lp": lp, "ids": ids,
                "done": done.to(torch.int32), "eos": ids.reshape(-1)[:2].contiguous()}
    if kind == "fork":
        t = _fork_tables(rng, case)
        book = _dev(np.concatenate([t["refs"], t["free"]]))
        return {"case": case, "table": _dev(t["table"]), "lens": _dev(t["lens"]), "parents": _dev(t["parents"]),
                "start": book, "book": book.clone(), "at": _dev([t["at"]])}
    p, moved = case["pages"], case["moved"]
    shape = (case["layers"], p, case["kv_heads"], 2, PART)
    pools = torch.randint(-2 ** 31, 2 ** 31, (math.prod(shape) // 2,), generator=g, device=DEV, dtype=torch.int32)
    pools.bitwise_and_(0x3FFF3FFF)                             # finite values
    pools = pools.view(torch.bfloat16).view(shape)
    perm = rng.permutation(p)
    return {"case": case, "all": pools, "pools": list(pools.unbind(0)), "src": _dev(perm[:moved]),
            "dst": _dev(perm[moved:2 * moved])}


# ----------------------------------------------------------------------------- plain forms
def _scores(x: torch.Tensor, tokens: torch.Tensor):
    """(the tokens' log-probabilities, log-probabilities, entropy, log of the sum of exponentials) of fp32 rows."""
    m = x.amax(-1, keepdim=True)
    lse = m + torch.log(torch.exp(x - m).sum(-1, keepdim=True))
    lp = x - lse
    p = torch.exp(lp)
    h = -torch.where(p > 0, p * lp, torch.zeros_like(p)).sum(-1)
    return lp.gather(1, tokens.long()[:, None])[:, 0], lp, h, lse[:, 0]


def _plain_logprobs(st: dict) -> dict:
    x, tok, n = st["logits"].float(), st["tokens"].long(), st["case"]["top"]
    idx = torch.arange(x.shape[1], device=DEV)
    xt = x.gather(1, tok[:, None])
    rank = ((x > xt) | ((x == xt) & (idx < tok[:, None]))).sum(-1).to(torch.int32)
    out, lp, h, _ = _scores(x, tok)
    res = {"logprob": out, "rank": rank, "entropy": h}
    if n:
        # one whole number a value: its place in the order of values, then the lower index
        bits = (x + 0.0).view(torch.int32).long()
        key = torch.where(bits < 0, -(bits & 0x7FFFFFFF), bits) * 2 ** 20 + (2 ** 20 - 1 - idx)
        ids = key.topk(n, -1).indices
        res |= {"top_ids": ids.to(torch.int32), "top_logprobs": lp.gather(1, ids)}
    return res


def _weights(packed: torch.Tensor, v: int, k: int, dtype=torch.float32) -> torch.Tensor:
    """The head's weights [V, K] from the packed bytes."""
    gp = k // 128
    w = packed.view(torch.int32).view(v // 16, gp * 288)
    nib = w[:, :gp * 256].reshape(-1, gp, 4, 16, 2, 2)         # block, pair, g, row, group, word
    e = torch.arange(8, device=DEV)
    q = (nib[..., None] >> (e % 2 * 16 + e // 2 * 4).to(torch.int32)) & 15
    sc = w[:, gp * 256:].contiguous().view(torch.bfloat16).to(dtype).view(-1, gp, 16, 2, 2)  # block, pair, row, s or b, group
    s, b = sc[..., 0, :], sc[..., 1, :]
    s, b = (t[:, :, None, :, :, None, None] for t in (s, b))
    full = q.to(dtype) * s + b                                 # block, pair, g, row, group, word, value
    return full.permute(0, 3, 1, 4, 2, 5, 6).reshape(v, k)


def _plain_head(st: dict) -> dict:
    case = st["case"]
    x = torch.matmul(st["x"].float(), _weights(st["head"], case["vocab"], case["hidden"]).t())
    out, _, h, lse = _scores(x, st["tokens"])
    return {"logprob": out, "entropy": h, "lse": lse}


def _plain_beams(st: dict) -> dict:
    gr, n, m = st["lp"].shape
    w, done, ids = st["case"]["width"], st["done"].bool(), st["ids"]
    first = torch.arange(m, device=DEV) == 0
    ended = done[:, :, None]
    score = torch.where(ended, st["scores"][:, :, None].expand(gr, n, m), st["scores"][:, :, None] + st["lp"])
    on = torch.where(ended, first, ids >= 0) & (score > -math.inf)
    score = torch.where(on, score, torch.full_like(score, -math.inf)).view(gr, n * m)
    token = torch.where(ended, torch.full_like(ids, -1), ids).view(gr, n * m)
    over = torch.nn.functional.pad(score, (0, max(0, w - n * m)), value=-math.inf)
    best, c = over.sort(dim=-1, descending=True, stable=True)
    best, c = best[:, :w], c[:, :w].clamp(max=n * m - 1)
    live = best > -math.inf
    tok = torch.where(live, token.gather(1, c).long(), -torch.ones_like(c))
    beam = c // m
    parent = torch.where(live, beam + n * torch.arange(gr, device=DEV)[:, None], -torch.ones_like(c))
    end = ~live | done.gather(1, beam) | (tok[:, :, None] == st["eos"].long()).any(-1)
    return {"parents": parent.to(torch.int32), "tokens": tok.to(torch.int32), "scores": best, "done": end.to(torch.int32)}


def _plain_fork(st: dict) -> dict:
    table, lens, par = st["table"].long(), st["lens"].long(), st["parents"].long()
    pages = st["case"]["pages"]
    st["book"].copy_(st["start"])
    refs, free = st["book"][:pages].long(), st["book"][pages:].long()
    at = st["at"].long()
    (s, w), n = table.shape, par.numel()
    i = torch.arange(n, device=DEV)
    live = (par >= 0) & (par < s)
    p = par.clamp(0, s - 1)
    held = (lens.clamp(min=0) + PAGE - 1) // PAGE
    first = torch.full((s + 1,), n, device=DEV).scatter_reduce(0, torch.where(live, p, s), i, "amin")[:s]
    last = (held - 1).clamp(min=0)
    tail = table.gather(1, last[:, None])[:, 0]
    open_ = (lens > 0) & (lens % PAGE != 0)
    need = live & open_[p] & ~((first[p] == i) & (refs[tail[p]] == 1))
    k = torch.cumsum(need, 0) - 1 + at
    got = need & (k < free.numel())
    refused = need & ~got
    dst = torch.where(got, free[k.clamp(0, free.numel() - 1)], torch.full_like(k, -1))
    src = torch.where(got, tail[p], torch.full_like(k, -1))
    on = live & ~refused
    j = torch.arange(w, device=DEV)
    new_len = torch.where(on, lens[p], torch.zeros_like(p))
    new = torch.where(j < ((new_len + PAGE - 1) // PAGE)[:, None], table[p], torch.zeros_like(table[p]))
    new = torch.where(got[:, None] & (j == last[p][:, None]), dst[:, None], new)
    # references: an entry's page gains one for each child that keeps it and loses its own
    count = torch.zeros(s + 1, dtype=torch.long, device=DEV).scatter_add(0, torch.where(on, p, s), torch.ones_like(p))[:s]
    keep = torch.zeros(s + 1, dtype=torch.long, device=DEV).scatter_add(0, torch.where(on & ~got, p, s), torch.ones_like(p))[:s]
    gain = torch.where(open_[:, None] & (j == last[:, None]), keep[:, None], count[:, None].expand(s, w)) - 1
    inside = j < held[:, None]
    refs = refs.scatter_add(0, table[inside], gain[inside])
    lost = torch.zeros(pages, dtype=torch.bool, device=DEV)
    lost[table[inside & (gain < 0)]] = True
    gone = torch.nonzero(lost & (refs == 0))[:, 0]             # ascending
    refs[dst[got]] = 1
    here = at + got.sum()
    back = here - gone.numel()
    free[back + torch.arange(gone.numel(), device=DEV)] = gone
    status = torch.cat([got.sum()[None], back, refused.sum()[None], torch.zeros_like(back)])
    return {"page_table": new.to(torch.int32), "lens": new_len.to(torch.int32), "src": src.to(torch.int32),
            "dst": dst.to(torch.int32), "status": status.to(torch.int32), "refs": refs.to(torch.int32),
            "free": free.to(torch.int32)}


# ----------------------------------------------------------------------------- one pass
def run(state: dict):
    case = state["case"]
    kind = case["kind"]
    if not own:
        if kind == "copy":
            dst, src = state["dst"].long(), state["src"].long()
            state["all"][:, dst] = state["all"][:, src]
            return state["all"]
        return {"logprobs": _plain_logprobs, "head": _plain_head, "beams": _plain_beams, "fork": _plain_fork}[kind](state)
    from jitengine_amd import ops

    if kind == "logprobs":
        r = ops.token_logprobs(state["logits"], state["tokens"], top=case["top"])
        res = {"logprob": r.logprob, "rank": r.rank, "entropy": r.entropy}
        if case["top"]:
            res |= {"top_ids": r.top_ids, "top_logprobs": r.top_logprobs}
        return res
    if kind == "head":
        if "packed" not in state:
            state["packed"] = ops.PackedQ4(state["head"], 1, case["vocab"], case["hidden"], False)
        r = ops.head_logprobs(state["x"], state["packed"], state["tokens"])
        return {"logprob": r.logprob, "entropy": r.entropy, "lse": r.lse}
    if kind == "beams":
        r = ops.beam_select(state["scores"], state["lp"], state["ids"], width=case["width"], done=state["done"],
                            eos=state["eos"])
        return {"parents": r.parents, "tokens": r.tokens, "scores": r.scores, "done": r.done}
    if kind == "fork":
        # (the counts and the list change in place: a pass begins with those of the step before)
        book, p = state["book"], case["pages"]
        book.copy_(state["start"])
        r = ops.pages_fork(state["table"], state["lens"], state["parents"], book[:p], book[p:], state["at"])
        return {"page_table": r.page_table, "lens": r.lens, "src": r.src, "dst": r.dst, "status": r.status,
                "refs": book[:p], "free": book[p:]}
    if "layers" not in state:
        state["layers"] = ops.pool_layers(state["pools"])
    ops.kv_copy_pages_layers(state["layers"], state["src"], state["dst"])
    return state["all"]


def work(case: dict) -> dict:
    kind = case["kind"]
    if kind == "logprobs":
        n, v = case["rows"], case["vocab"]
        return {"bytes": 2 * n * v + 16 * n + 8 * n * case["top"], "flops": 6 * n * v}
    if kind == "head":
        n, v, k = case["rows"], case["vocab"], case["hidden"]
        return {"bytes": v * k * 9 // 16 + 2 * n * k + 16 * n, "flops": 2 * n * v * k + 6 * n * v}
    if kind == "beams":
        gr, n, m = case["groups"], case["beams"], case["alts"]
        return {"bytes": gr * (8 * n * m + 8 * n + 16 * case["width"]), "flops": gr * n * m}
    if kind == "fork":
        # pages of a mean sequence, read from its parent's row and written to its own, and each page's count
        s = case["groups"] * case["beams"]
        held = (3 * case["prompt"] // 4 + case["fresh"] // 2) // PAGE + 1
        return {"bytes": s * (16 * held + 20), "flops": 0}
    return {"bytes": 2 * case["layers"] * case["moved"] * case["kv_heads"] * 2 * PART * 2, "flops": 0}


# ----------------------------------------------------------------------------- 64 bits
def _exact_rows(x: torch.Tensor, tok: torch.Tensor):
    """log softmax of the tokens, entropy and log of the sum of exponentials of rows, by the definitions."""
    lse = torch.logsumexp(x, -1)
    p = torch.exp(x - lse[:, None])
    h = torch.special.entr(p).sum(-1)
    return x[torch.arange(x.shape[0], device=DEV), tok.long()] - lse, h, lse


def exact(case: dict, seed: int):
    kind = case["kind"]
    if kind == "fork":
        return None                                            # whole numbers alone
    st = prepare(case, seed)
    if kind == "copy":
        pools = st["all"].double()
        return pools.index_copy(1, st["dst"].long(), pools.index_select(1, st["src"].long()))
    if kind == "logprobs":
        parts = [_exact_rows(x.double(), t) for x, t in zip(st["logits"].split(256), st["tokens"].split(256))]
        lp, h, lse = (torch.cat(t) for t in zip(*parts))
        res = {"logprob": lp, "rank": None, "entropy": h}
        if case["top"]:
            best = torch.cat([x.double().topk(case["top"], -1).values for x in st["logits"].split(256)])
            res |= {"top_ids": None, "top_logprobs": best - lse[:, None]}
        return res
    if kind == "head":
        v, k = case["vocab"], case["hidden"]
        rows = []
        for a in range(0, v, 16384):                           # weights a slice of the vocabulary at a time
            n = min(16384, v - a)
            raw = st["head"].view(torch.int16).view(v // 16, -1)[a // 16:(a + n) // 16].int() & 0xFFFF
            nib = raw[:, :k * 4].reshape(n // 16, k // 128, 64, 8)
            tile = torch.stack([(nib >> (4 * i)) & 15 for i in range(4)], -1)  # ..., lane, half word, place
            tile = tile.view(n // 16, k // 128, 4, 16, 2, 2, 2, 4).transpose(-1, -2)  # g, row, group, word, place, odd
            q = tile.permute(0, 3, 1, 4, 2, 5, 6, 7).reshape(n, k // 64, 64).double()
            sb = (raw[:, k * 4:] << 16).view(torch.float32).view(n // 16, k // 128, 16, 2, 2).permute(0, 2, 3, 1, 4)
            sb = sb.reshape(n // 16, 16, 2, k // 64).double()
            w = q * sb[:, :, 0].reshape(n, -1, 1) + sb[:, :, 1].reshape(n, -1, 1)
            rows.append(st["x"].double() @ w.view(n, k).t())
        x = torch.cat(rows, 1)
        lp, h, lse = _exact_rows(x, st["tokens"])
        return {"logprob": lp, "entropy": h, "lse": lse}
    d = st["done"].bool()[..., None]
    c = torch.where(d, st["scores"].double()[..., None].expand(st["lp"].shape), st["scores"].double()[..., None] + st["lp"].double())
    c[..., 1:] = torch.where(d, torch.full_like(c[..., 1:], -math.inf), c[..., 1:])
    c = c.flatten(1)
    w = case["width"]
    best = torch.full((c.shape[0], w), -math.inf, dtype=torch.float64, device=DEV)
    k = min(w, c.shape[1])
    best[:, :k] = c.topk(k, -1).values
    return {"parents": None, "tokens": None, "scores": best, "done": None}
