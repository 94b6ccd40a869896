"""The 8-bit KV cache and its tables as calls that can be timed and compared: each operator in its plain form
(elementary torch operations, 32 bits) and as a program calls it of this framework.

A cache page holds 16 tokens.  Each (page, kv head) has one record of 4,224 bytes:

  [0, 2048)     K codes, [2][4][16 slots][16]: index (i, g, slot, x) is dim 64 i + 16 g + x;
  [2048, 4096)  V codes, [2][4][16][4][4]: index (q, g, r, c, j) is dim 16 (4 q + c) + r of slot 4 g + j;
  [4096, 4224)  32 fp32 scales: K of slots 0 .. 15, then V of slots 0 .. 15.

Codes are e4m3 (largest magnitude 448).  A token's K (and V) of one kv head has one scale, the power of two 2^e with
e = E - 8, or E - 7 where the largest magnitude (1 + m) 2^E has m > 0.75; a row of zeros has scale 1.

Kinds of case (geometry of `jitengine_amd.model.MoEConfig` unless the heads are given):

  tables   page tables, positions and slots of a step from its sequences' lengths (`ops.step_tables`);
  write    q/k norm, RoPE and the cache write of a step's raw q/k/v rows (`ops.qk_norm_rope_append_kv8`), or the
           write alone of given k and v (`ops.kv8_append_paged`);
  decode   attention of single tokens over the cache (`ops.paged_decode_attention_kv8`);
  prompt   causal attention of prompt chunks of different lengths (`ops.paged_prefill_attention_kv8`).
"""

from __future__ import annotations

import math
import random

import numpy as np
import torch

own = False

DEV = "cuda"
PAGE, DH, REC = 16, 128, 4224
EPS, THETA = 1e-6, 1e6
SCALE = DH ** -0.5


# ----------------------------------------------------------------------------- the cases
def listed() -> list:
    return [
        # a lone sequence's step: the smallest tables call, latency alone
        {"name": "tables_1", "kind": "tables", "seqs": 1, "chunks": 0, "rows": 1, "ctx": 4096, "seed": 1},
        # a mixed step: four prompt chunks and 60 decode rows
        {"name": "tables_mixed_2108", "kind": "tables", "seqs": 64, "chunks": 4, "rows": 2108, "ctx": 16384, "seed": 2},
        # a large deployment's step: 1,024 sequences, eight of them in their prompts
        {"name": "tables_1024_seqs", "kind": "tables", "seqs": 1024, "chunks": 8, "rows": 9208, "ctx": 8192, "seed": 3},
        # the write of a decode step's 32 rows
        {"name": "write_decode_32", "kind": "write", "rows": 32, "H": 32, "Hkv": 4, "ctx": 32768, "raw": False, "seed": 4},
        # the write of a mixed step's rows
        {"name": "write_mixed_2108", "kind": "write", "rows": 2108, "H": 32, "Hkv": 4, "ctx": 16384, "raw": False,
         "seed": 5},
        # the write alone, k and v already made, of as many kv heads as query heads
        {"name": "write_raw_1001", "kind": "write", "rows": 1001, "H": 16, "Hkv": 16, "ctx": 8192, "raw": True, "seed": 6},
        # one user, an ordinary context: the smallest attention call
        {"name": "decode_1x4096", "kind": "decode", "batch": 1, "lo": 4096, "hi": 4096, "H": 32, "Hkv": 4, "seed": 7},
        # a serving batch of ragged contexts
        {"name": "decode_32_ragged", "kind": "decode", "batch": 32, "lo": 128, "hi": 32768, "H": 32, "Hkv": 4, "seed": 8},
        # one user at the longest context
        {"name": "decode_1x262144", "kind": "decode", "batch": 1, "lo": 262144, "hi": 262144, "H": 32, "Hkv": 4, "seed": 9},
        # a short prompt's only chunk, odd in length
        {"name": "prompt_77", "kind": "prompt", "chunks": 1, "rows": 77, "ctx": 0, "H": 32, "Hkv": 4, "seed": 10},
        # the engine's prompt chunks of four sequences of different lengths
        {"name": "prompt_4_ragged", "kind": "prompt", "chunks": 4, "rows": 1500, "ctx": 8192, "H": 32, "Hkv": 4, "seed": 11},
        # one long chunk deep into its prompt
        {"name": "prompt_2048_deep", "kind": "prompt", "chunks": 1, "rows": 2048, "ctx": 8192, "H": 32, "Hkv": 4, "seed": 12},
    ]


def _log(rng: random.Random, lo: int, hi: int) -> int:
    return max(lo, min(hi, round(math.exp(rng.uniform(math.log(lo), math.log(hi + 1))))))


def draw(rng: random.Random) -> dict:
    """A case of the ranges the listed ones stand for."""
    kind = rng.choice(["tables", "write", "write", "decode", "decode", "decode", "prompt", "prompt"])
    seed = rng.randrange(1 << 20)
    if kind == "tables":
        seqs = _log(rng, 1, 1024)
        chunks = min(seqs, rng.choice([0, 1, 2, 4, 8]))
        rows = seqs - chunks + (_log(rng, chunks, 1024 * chunks) if chunks else 0)
        return {"kind": kind, "seqs": seqs, "chunks": chunks, "rows": rows, "ctx": _log(rng, 16, 16384), "seed": seed}
    if kind == "write":
        h, hkv = rng.choice([(32, 4), (32, 4), (16, 16), (8, 2), (64, 4), (12, 4)])
        return {"kind": kind, "rows": _log(rng, 1, 2108), "H": h, "Hkv": hkv, "ctx": _log(rng, 16, 262144),
                "raw": rng.random() < 0.3, "seed": seed}
    if kind == "decode":
        h, hkv = rng.choice([(32, 4), (32, 4), (16, 16), (8, 2), (64, 4), (12, 4)])
        batch = _log(rng, 1, 64)
        hi = _log(rng, 1, min(262144, 1048576 // (batch * hkv)))
        return {"kind": kind, "batch": batch, "lo": _log(rng, 1, hi), "hi": hi, "H": h, "Hkv": hkv, "seed": seed}
    h, hkv = rng.choice([(32, 4), (32, 4), (16, 16), (8, 2), (32, 8)])
    chunks = rng.choice([1, 1, 2, 4])
    return {"kind": kind, "chunks": chunks, "rows": max(chunks, _log(rng, 1, 2048 // chunks)), "ctx": _log(rng, 1, 8192), "H": h,
            "Hkv": hkv, "seed": seed}


def _lens(case: dict) -> np.ndarray:
    """Keys of each decode sequence (log-uniform in [lo, hi])."""
    rng = np.random.default_rng(case["seed"])
    lo, hi, n = case["lo"], case["hi"], case["batch"]
    ln = np.round(np.exp(rng.uniform(np.log(lo), np.log(hi), n))) if hi > lo else np.full(n, lo)
    return np.clip(ln, lo, hi).astype(np.int32)


def _split(rng, total: int, parts: int) -> np.ndarray:
    """total rows in `parts` chunks of different lengths, each at least one row."""
    cuts = np.sort(rng.choice(np.arange(1, total), parts - 1, replace=False)) if parts > 1 else np.zeros(0, np.int64)
    return np.diff(np.concatenate([[0], cuts, [total]])).astype(np.int64)


def _chunks(case: dict) -> list:
    """(sequence, positions before the chunk, rows) of each prompt chunk; contexts uniform in [0, ctx]."""
    rng = np.random.default_rng(case["seed"])
    n = case["chunks"]
    lens = _split(rng, case["rows"], n)
    ctx = rng.integers(0, case["ctx"] + 1, n) if n > 1 else np.array([case["ctx"]])
    return [(i, int(ctx[i]), int(lens[i])) for i in range(n)]


def _step(case: dict):
    """(positions before, new rows) of each sequence of a step: the prompt chunks first, then decode rows."""
    rng = np.random.default_rng(case["seed"])
    n, c = case["seqs"], case["chunks"]
    new = np.ones(n, np.int64)
    if c:
        new[:c] = _split(rng, case["rows"] - (n - c), c)
    ctx = rng.integers(0, case["ctx"] + 1, n)
    ctx[c:] = np.maximum(ctx[c:], 1)
    return ctx.astype(np.int64), new


# ----------------------------------------------------------------------------- inputs
def _gen(seed: int) -> torch.Generator:
    g = torch.Generator(device=DEV)
    g.manual_seed(int(seed))
    return g


def _rand(g, *shape) -> torch.Tensor:
    return torch.randn(shape, generator=g, device=DEV)


def _quantise(x: torch.Tensor):
    """x [..., 128] fp32 -> (codes as float8 [..., 128], scales fp32 [...]) of the cache's definition."""
    amax = x.abs().amax(-1)
    m, e = torch.frexp(amax)                             # amax = m 2^e, m in [0.5, 1)
    e = (e - 9 + (m > 0.875).int()).clamp(-100, 118)
    scale = torch.where(amax > 0, ((e + 127) << 23).view(torch.float32), torch.ones_like(amax))
    return (x / scale[..., None]).clamp(-448, 448).to(torch.float8_e4m3fn), scale


def _records(k: torch.Tensor, v: torch.Tensor) -> torch.Tensor:
    """k, v [pages, Hkv, 16, 128] fp32 -> records [pages, Hkv, 4224] uint8."""
    p, h = k.shape[:2]
    kc, ks = _quantise(k)
    vc, vs = _quantise(v)
    kc = kc.view(torch.uint8).view(p, h, 16, 2, 4, 16).permute(0, 1, 3, 4, 2, 5).reshape(p, h, 2048)
    vc = vc.view(torch.uint8).view(p, h, 4, 4, 2, 4, 16).permute(0, 1, 4, 2, 6, 5, 3).reshape(p, h, 2048)
    sc = torch.cat([ks, vs], -1).contiguous().view(torch.uint8)
    return torch.cat([kc, vc, sc], -1).contiguous()


def _pool(g, pages: int, hkv: int) -> torch.Tensor:
    """A cache as earlier steps left it: normed keys with loud and quiet channels, values of uneven tokens."""
    out = torch.empty((pages, hkv, REC), dtype=torch.uint8, device=DEV)
    wk = 1.0 + 0.3 * _rand(g, hkv, 1, DH)
    for p0 in range(0, pages, 4096):
        n = min(4096, pages - p0)
        k = _rand(g, n, hkv, PAGE, DH) * wk
        v = _rand(g, n, hkv, PAGE, DH) * torch.exp(0.7 * _rand(g, n, hkv, PAGE, 1))
        out[p0:p0 + n] = _records(k, v)
    return out


def _table(rng, need: np.ndarray, spare: int):
    """Page tables over a random permutation of the pool's pages: (table [S, W] int32, pages in the pool)."""
    total = int(need.sum())
    perm = rng.permutation(total + spare).astype(np.int32)
    t = np.zeros((len(need), max(1, int(need.max(initial=1)))), np.int32)
    at = np.concatenate([[0], np.cumsum(need)])
    mask = np.arange(t.shape[1])[None] < need[:, None]
    t[mask] = perm[:total]
    return t, total + spare, perm[total:], at


def _inv_freq() -> torch.Tensor:
    f = float(THETA) ** (-np.arange(0, DH, 2, dtype=np.float64) / DH)
    return torch.from_numpy(f.astype(np.float32)).to(DEV)


def _dev(a, dtype=np.int32) -> torch.Tensor:
    return torch.from_numpy(np.ascontiguousarray(np.asarray(a).astype(dtype))).to(DEV)


def prepare(case: dict, seed: int) -> dict:
    g = _gen(seed)
    rng = np.random.default_rng([seed, case["seed"]])
    kind = case["kind"]
    if kind == "tables":
        ctx, new = _step(case)
        have, tot = -(-ctx // PAGE), -(-(ctx + new) // PAGE)
        t, pages, _, _ = _table(rng, have, 0)
        table = np.zeros((len(ctx), int(tot.max()) + 3), np.int32)
        table[:, :t.shape[1]] = t
        # the free list covers the step, or (every fourth seed) falls short for the last sequences
        need = int((tot - have).sum())
        free = pages + rng.permutation(max(1, need // 2 if seed % 4 == 3 else need + 64))
        return {"case": case, "ctx": _dev(ctx), "new": _dev(new), "table": _dev(table), "free": _dev(free),
                "rows": case["rows"]}
    h, hkv = case["H"], case["Hkv"]
    if kind == "write":
        n = case["rows"]
        pos = rng.integers(0, case["ctx"], n)
        pages = n // 8 + 2
        slots = rng.permutation(pages * PAGE)[:n]
        st = {"case": case, "pool": _pool(g, pages, hkv), "pos": _dev(pos), "slots": _dev(slots)}
        if case["raw"]:
            st["k"] = _rand(g, n, hkv, DH).to(torch.bfloat16)
            st["v"] = (_rand(g, n, hkv, DH) * torch.exp(_rand(g, n, hkv, 1))).to(torch.bfloat16)
        else:
            st["qkv"] = (2.0 * _rand(g, n, (h + 2 * hkv) * DH)).to(torch.bfloat16)
            st["q_norm"] = (1.0 + 0.3 * _rand(g, DH)).to(torch.bfloat16)
            st["k_norm"] = (1.0 + 0.3 * _rand(g, DH)).to(torch.bfloat16)
            st["inv_freq"] = _inv_freq()
        return st
    if kind == "decode":
        lens = _lens(case)
        table, pages, _, _ = _table(rng, -(-lens.astype(np.int64) // PAGE), 4)
        return {"case": case, "pool": _pool(g, pages, hkv), "table": _dev(table), "lens": _dev(lens),
                "max_len": int(lens.max()), "q": (1.5 * _rand(g, len(lens), h, DH)).to(torch.bfloat16)}
    chunks = _chunks(case)
    keys = np.array([c + n for _, c, n in chunks], np.int64)
    table, pages, _, _ = _table(rng, -(-keys // PAGE), 4)
    st = {"case": case, "chunks": chunks, "pool": _pool(g, pages, hkv), "table": _dev(table),
          "q": (1.5 * _rand(g, case["rows"], h, DH)).to(torch.bfloat16)}
    # where each row sits in a [chunks, longest chunk] grid, and each chunk's context
    lens = np.array([n for _, _, n in chunks])
    st["longest"] = int(lens.max())
    st["at"] = _dev(np.concatenate([i * int(lens.max()) + np.arange(n) for i, n in enumerate(lens)]), np.int64)
    st["ctx"] = _dev([c for _, c, _ in chunks], np.int64)
    if own:
        from jitengine_amd import ops

        st["plan"] = ops.prefill_plan(chunks, h, hkv, DEV)
    return st


# ----------------------------------------------------------------------------- plain forms
def _read(pool: torch.Tensor, table: torch.Tensor):
    """The cache's values through page tables [S, W]: k, v fp32 [S, Hkv, 16 W, 128]."""
    rec = pool[table.long()]                             # [S, W, Hkv, 4224]
    s, w, h = rec.shape[:3]
    sc = rec[..., 4096:].contiguous().view(torch.float32)
    c = rec[..., :4096].contiguous().view(torch.float8_e4m3fn).float()
    k = c[..., :2048].view(s, w, h, 2, 4, 16, 16).permute(0, 2, 1, 5, 3, 4, 6).reshape(s, h, w * 16, DH)
    v = c[..., 2048:].view(s, w, h, 2, 4, 16, 4, 4).permute(0, 2, 1, 4, 7, 3, 6, 5).reshape(s, h, w * 16, DH)
    ks = sc[..., :16].permute(0, 2, 1, 3).reshape(s, h, w * 16, 1)
    vs = sc[..., 16:].permute(0, 2, 1, 3).reshape(s, h, w * 16, 1)
    return k * ks, v * vs


def _softmax(s: torch.Tensor) -> torch.Tensor:
    p = torch.exp(s - s.amax(-1, keepdim=True))
    return p / p.sum(-1, keepdim=True)


def _plain_tables(st: dict) -> dict:
    ctx, new, table, free, rows = st["ctx"].long(), st["new"].long(), st["table"], st["free"], st["rows"]
    have, tot = (ctx + PAGE - 1) // PAGE, (ctx + new + PAGE - 1) // PAGE
    end = torch.cumsum(new, 0)
    start = end - new
    fits = (tot <= table.shape[1]) & (end <= rows)
    need = torch.where(fits, tot - have, torch.zeros_like(tot))
    cum = torch.cumsum(need, 0)
    served = fits & ((need == 0) | (cum <= free.numel()))
    r = torch.arange(rows, device=DEV)
    seq = torch.searchsorted(end, r, right=True)
    live = seq < ctx.numel()
    b = seq.clamp(max=ctx.numel() - 1)
    pos = torch.where(live, ctx[b] + r - start[b], torch.zeros_like(r))
    pi = pos // PAGE
    fresh = pi >= have[b]
    ok = live & served[b]
    at = (cum - need)[b] + pi - have[b]
    page = torch.where(fresh, free[at.clamp(0, free.numel() - 1)].long(),
                       table[b, pi.clamp(max=table.shape[1] - 1)].long())
    slots = torch.where(ok, page * PAGE + pos % PAGE, torch.full_like(pos, -1))
    put = ok & fresh & ((pos % PAGE == 0) | (pos == ctx[b]))
    flat = torch.where(put, b * table.shape[1] + pi, torch.full_like(pi, table.numel()))
    grown = torch.cat([table.reshape(-1), table.new_zeros(1)])
    grown[flat] = page.to(torch.int32)
    return {"row_start": torch.cat([start, end[-1:]]).int(), "row_seq": torch.where(live, seq, torch.full_like(seq, -1)).int(),
            "pos": pos.int(), "slots": slots.int(), "lens": torch.where(served, ctx + new, ctx).int(),
            "status": torch.stack([end[-1], (need * served).sum(), (~served).sum(), torch.zeros_like(end[-1])]).int(),
            "page_table": grown[:-1].reshape(table.shape)}


def _plain_norm_rope(x: torch.Tensor, w: torch.Tensor, cos: torch.Tensor, sin: torch.Tensor) -> torch.Tensor:
    x = x.float()
    y = x * torch.rsqrt(x.square().mean(-1, keepdim=True) + EPS) * w.float()
    a, b = y[..., :64], y[..., 64:]
    return torch.cat([a * cos - b * sin, a * sin + b * cos], -1)


def _plain_write(st: dict) -> dict:
    case, pool, slots = st["case"], st["pool"], st["slots"].long()
    h, hkv = case["H"], case["Hkv"]
    out = {}
    if case["raw"]:
        k, v = st["k"].float(), st["v"].float()
    else:
        x = st["qkv"].view(-1, h + 2 * hkv, DH)
        ang = st["pos"].double()[:, None] * st["inv_freq"].double()[None]
        cos, sin = torch.cos(ang).float()[:, None], torch.sin(ang).float()[:, None]
        out["q"] = _plain_norm_rope(x[:, :h], st["q_norm"], cos, sin).to(torch.bfloat16)
        k = _plain_norm_rope(x[:, h:h + hkv], st["k_norm"], cos, sin)
        v = x[:, h + hkv:].float()
    page, slot = slots // PAGE, slots % PAGE
    kc, ks = _quantise(k)
    vc, vs = _quantise(v)
    d = torch.arange(DH, device=DEV)
    n = torch.arange(hkv, device=DEV)
    # byte of (slot, dim) in the K and V parts of a record
    kat = (d // 64) * 1024 + (d // 16 % 4) * 256 + d % 16 + slot[:, None] * 16
    vat = 2048 + (d // 64) * 1024 + (d % 16) * 16 + (d // 16 % 4) * 4 + ((slot // 4) * 256 + slot % 4)[:, None]
    pool[page[:, None, None], n[None, :, None], kat[:, None, :]] = kc.view(torch.uint8)
    pool[page[:, None, None], n[None, :, None], vat[:, None, :]] = vc.view(torch.uint8)
    sc = pool[..., 4096:].view(torch.float32)
    sc[page[:, None], n[None], slot[:, None]] = ks
    sc[page[:, None], n[None], 16 + slot[:, None]] = vs
    return out


def _plain_decode(st: dict) -> torch.Tensor:
    q, lens = st["q"], st["lens"].long()
    b, h = q.shape[:2]
    k, v = _read(st["pool"], st["table"])
    hkv, n = k.shape[1:3]
    s = torch.matmul(q.float().view(b, hkv, h // hkv, DH), k.transpose(2, 3).contiguous()) * SCALE
    keep = torch.arange(n, device=DEV) < lens[:, None]
    s = torch.where(keep[:, None, None], s, torch.full_like(s, -math.inf))
    return torch.matmul(_softmax(s), v).view(b, h, DH).to(torch.bfloat16)


def _plain_prompt(st: dict) -> torch.Tensor:
    q, at, m = st["q"], st["at"], st["longest"]
    h = q.shape[1]
    k, v = _read(st["pool"], st["table"])
    c, hkv, n = k.shape[:3]
    grid = q.new_zeros((c * m, h, DH), dtype=torch.float32)
    grid[at] = q.float()
    g = h // hkv
    x = grid.view(c, m, hkv, g, DH).permute(0, 2, 3, 1, 4).reshape(c, hkv, g * m, DH)
    s = torch.matmul(x, k.transpose(2, 3).contiguous()) * SCALE
    pos = (st["ctx"][:, None] + torch.arange(m, device=DEV)).repeat(1, g)
    s.masked_fill_((torch.arange(n, device=DEV) > pos[..., None])[:, None], -math.inf)
    o = torch.matmul(_softmax(s), v).view(c, hkv, g, m, DH).permute(0, 3, 1, 2, 4).reshape(c * m, h, DH)
    return o[at].to(torch.bfloat16)


# ----------------------------------------------------------------------------- one pass
def _cache(pool: torch.Tensor) -> dict:
    """The cache as the values it holds: e4m3 codes and their scales."""
    return {"codes": pool[..., :4096].view(torch.float8_e4m3fn), "scales": pool[..., 4096:].view(torch.float32)}


def run(state: dict):
    case = state["case"]
    kind = case["kind"]
    if not own:
        if kind == "tables":
            return _plain_tables(state)
        if kind == "write":
            out = _plain_write(state)
            return {**out, **_cache(state["pool"])}
        return _plain_decode(state) if kind == "decode" else _plain_prompt(state)
    from jitengine_amd import ops

    if kind == "tables":
        t = ops.step_tables(state["ctx"], state["new"], state["table"], state["rows"], free=state["free"])
        return {"row_start": t.row_start, "row_seq": t.row_seq, "pos": t.pos, "slots": t.slots, "lens": t.lens,
                "status": t.status, "page_table": state["table"]}
    if kind == "write":
        pool = state["pool"]
        if case["raw"]:
            ops.kv8_append_paged(pool, state["k"], state["v"], state["slots"])
            return _cache(pool)
        q = ops.qk_norm_rope_append_kv8(state["qkv"], case["H"], case["Hkv"], state["q_norm"], state["k_norm"], EPS,
                                        state["inv_freq"], state["pos"], state["slots"], pool)
        return {"q": q, **_cache(pool)}
    if kind == "decode":
        return ops.paged_decode_attention_kv8(state["q"], state["pool"], state["table"], state["lens"],
                                              state["max_len"], SCALE)
    return ops.paged_prefill_attention_kv8(state["q"], state["pool"], state["table"], state["plan"], SCALE)


def work(case: dict) -> dict:
    kind = case["kind"]
    if kind == "tables":
        ctx, new = _step(case)
        pages = int((-(-(ctx + new) // PAGE) + -ctx // PAGE).sum())
        return {"bytes": 8 * len(ctx) + 8 * pages + 12 * case["rows"] + 8 * len(ctx), "flops": 0}
    h, hkv = case["H"], case["Hkv"]
    token = 2 * hkv * (DH + 4)  # bytes of one position in the cache
    if kind == "write":
        n = case["rows"]
        if case["raw"]:
            return {"bytes": n * (4 * hkv * DH + token + 4), "flops": 0}
        return {"bytes": n * (2 * (h + 2 * hkv) * DH + 2 * h * DH + token + 8), "flops": n * (h + hkv) * DH * 10}
    if kind == "decode":
        keys = int(_lens(case).astype(np.int64).sum())
        return {"bytes": keys * token + 4 * case["batch"] * h * DH + keys // 4, "flops": 4 * keys * h * DH}
    pairs = sum(n * c + n * (n + 1) // 2 for _, c, n in _chunks(case))
    keys = sum(c + n for _, c, n in _chunks(case))
    return {"bytes": keys * token + 4 * case["rows"] * h * DH + keys // 4, "flops": 4 * pairs * h * DH}


# ----------------------------------------------------------------------------- 64 bits
def _e4m3_values() -> torch.Tensor:
    """The 256 values of e4m3 from its definition: sign, 4 exponent bits of bias 7, 3 mantissa bits."""
    c = np.arange(256)
    e, m = (c >> 3) & 15, c & 7
    v = np.where(e > 0, (1 + m / 8) * 2.0 ** (e - 7), m / 8 * 2.0 ** -6)
    v = np.where((c & 127) == 127, np.nan, v)
    return torch.from_numpy(np.where(c >= 128, -v, v)).to(DEV)


def _exact_codes(x: torch.Tensor, lut: torch.Tensor):
    """(codes uint8, scales) of rows x [..., 128] in 64 bits: the nearest e4m3 value, ties to the even code."""
    amax = x.abs().amax(-1)
    e = torch.floor(torch.log2(amax.clamp_min(1e-300)))
    e = torch.where(torch.exp2(e) > amax, e - 1, e)
    e = torch.where(torch.exp2(e + 1) <= amax, e + 1, e)
    e = torch.where(amax > 1.75 * torch.exp2(e), e - 7, e - 8).clamp(-100, 118)
    scale = torch.where(amax > 0, torch.exp2(e), torch.ones_like(e))
    y = (x / scale[..., None]).clamp(-448, 448)
    mag = lut[:127].contiguous()                         # ascending
    hi = torch.searchsorted(mag, y.abs().contiguous()).clamp(max=126)
    lo = (hi - 1).clamp(min=0)
    dl, dh = y.abs() - mag[lo], mag[hi] - y.abs()
    c = torch.where(dl < dh, lo, torch.where(dl > dh, hi, torch.where(lo % 2 == 0, lo, hi)))
    return (c + 128 * torch.signbit(y)).to(torch.uint8), scale


def _exact_kv(pool: torch.Tensor, pages: torch.Tensor, head: int, lut: torch.Tensor):
    """k, v in 64 bits of one kv head's pages, [16 n, 128]."""
    rec = pool[pages.long(), head]
    sc = rec[:, 4096:].contiguous().view(torch.float32).double()
    c = lut[rec[:, :4096].long()]
    k = torch.einsum("pigsx->psigx", c[:, :2048].reshape(-1, 2, 4, 16, 16)).reshape(-1, 16, DH) * sc[:, :16, None]
    v = torch.einsum("pqgrcj->pgjqcr", c[:, 2048:].reshape(-1, 2, 4, 16, 4, 4)).reshape(-1, 16, DH) * sc[:, 16:, None]
    return k.reshape(-1, DH), v.reshape(-1, DH)


def _exact_attention(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, last: torch.Tensor) -> torch.Tensor:
    """q [n, 128], row i over keys 0 .. last[i]."""
    out = torch.empty((q.shape[0], DH), dtype=torch.float64, device=DEV)
    kt = k.t().contiguous()
    for i in range(0, q.shape[0], 4096):
        s = (q[i:i + 4096].double() @ kt) * SCALE
        s.masked_fill_(torch.arange(k.shape[0], device=DEV)[None] > last[i:i + 4096, None], -math.inf)
        p = torch.exp(s - s.max(-1, keepdim=True).values)
        out[i:i + 4096] = (p @ v) / p.sum(-1, keepdim=True)
    return out


def exact(case: dict, seed: int):
    st = prepare(case, seed)
    kind = case["kind"]
    if kind == "tables":  # whole numbers, which both sides have to give alike
        return None
    h, hkv, lut = case["H"], case["Hkv"], _e4m3_values()
    if kind == "write":
        out = {}
        if case["raw"]:
            k, v = st["k"].double(), st["v"].double()
        else:
            x = st["qkv"].double().view(-1, h + 2 * hkv, DH)
            rot = torch.polar(torch.ones((case["rows"], 1, 64), dtype=torch.float64, device=DEV),
                              (st["pos"].double()[:, None] * st["inv_freq"].double())[:, None])

            def head(y, w):
                y = y / torch.sqrt((y * y).sum(-1, keepdim=True) / DH + EPS) * w.double()
                z = torch.complex(y[..., :64].contiguous(), y[..., 64:].contiguous()) * rot
                return torch.cat([z.real, z.imag], -1)

            out["q"] = head(x[:, :h], st["q_norm"])
            k, v = head(x[:, h:h + hkv], st["k_norm"]), x[:, h + hkv:]
        codes = lut[st["pool"][..., :4096].long()]
        scales = st["pool"][..., 4096:].contiguous().view(torch.float32).double()
        (kc, ks), (vc, vs) = _exact_codes(k, lut), _exact_codes(v, lut)
        page, slot = st["slots"].long() // PAGE, st["slots"].long() % PAGE
        kk = codes[..., :2048].reshape(-1, hkv, 2, 4, 16, 16)
        vv = codes[..., 2048:].reshape(-1, hkv, 2, 4, 16, 4, 4)
        kk[page, :, :, :, slot] = lut[kc.long()].view(-1, hkv, 2, 4, 16)
        vv[page, :, :, slot // 4, :, :, slot % 4] = lut[vc.long()].view(-1, hkv, 2, 4, 16).transpose(3, 4)
        scales[page, :, slot], scales[page, :, 16 + slot] = ks, vs
        p = codes.shape[0]
        return {**out, "codes": torch.cat([kk.reshape(p, hkv, 2048), vv.reshape(p, hkv, 2048)], -1), "scales": scales}
    g, out = h // hkv, torch.empty(st["q"].shape, dtype=torch.float64, device=DEV)
    if kind == "decode":
        for b, n in enumerate(_lens(case).tolist()):
            for j in range(hkv):
                k, v = _exact_kv(st["pool"], st["table"][b, :-(-n // PAGE)], j, lut)
                last = torch.full((g,), n - 1, device=DEV)
                out[b, j * g:(j + 1) * g] = _exact_attention(st["q"][b, j * g:(j + 1) * g], k[:n], v[:n], last)
        return out
    row = 0
    for c, ctx, n in st["chunks"]:
        for j in range(hkv):
            k, v = _exact_kv(st["pool"], st["table"][c, :-(-(ctx + n) // PAGE)], j, lut)
            x = st["q"][row:row + n, j * g:(j + 1) * g].reshape(n * g, DH)
            last = ctx + torch.arange(n, device=DEV).repeat_interleave(g)
            out[row:row + n, j * g:(j + 1) * g] = _exact_attention(x, k, v, last).view(n, g, DH)
        row += n
    return out
