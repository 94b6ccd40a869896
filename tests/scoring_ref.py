"""Plain 64-bit and whole-number implementations of the scoring and continuation operators, for their tests."""

from __future__ import annotations

import math

import numpy as np
import torch

PAGE = 16


def rows_ref(x: torch.Tensor, tokens: torch.Tensor | None, top: int):
    """(logprob, rank, entropy, top_ids, top_logprobs) of logits [B, V] by the definitions, fp64 on the CPU."""
    x = x.detach().cpu().double()
    B, V = x.shape
    tk = torch.zeros((B, 0), dtype=torch.int64) if tokens is None else tokens.detach().cpu().long().reshape(B, -1)
    lp, rank = torch.zeros(tk.shape, dtype=torch.float64), torch.full(tk.shape, -1, dtype=torch.int64)
    ent = torch.zeros(B, dtype=torch.float64)
    ids, tlp = torch.full((B, top), -1, dtype=torch.int64), torch.full((B, top), math.nan, dtype=torch.float64)
    for b in range(B):
        r = x[b]
        bad = bool(torch.isnan(r).any() or (r == math.inf).any())
        m = r.max()
        if bad:
            row, ent[b] = torch.full_like(r, math.nan), math.nan
            row[r == -math.inf] = math.nan
        elif m == -math.inf:
            row = r.clone()
        else:
            e = torch.exp(r - m)
            row = (r - m) - torch.log(e.sum())
            p = e / e.sum()
            ent[b] = -(p[p > 0] * row[p > 0]).sum()
        ok = torch.nonzero(~torch.isnan(r))[:, 0]
        order = ok[torch.sort(-r[ok], stable=True).indices]
        place = torch.full((V,), -1, dtype=torch.int64)
        place[order] = torch.arange(order.numel())
        for q in range(tk.shape[1]):
            t = int(tk[b, q])
            if 0 <= t < V:
                lp[b, q], rank[b, q] = row[t], place[t]
        n = min(top, order.numel())
        ids[b, :n] = order[:n]
        tlp[b, :n] = row[order[:n]]
    if tokens is not None:
        lp, rank = lp.view(tokens.shape), rank.view(tokens.shape)
    return lp, rank, ent, ids, tlp


def beams_ref(scores, lp, ids, width, done=None, eos=()):
    """beam_select by sorting each group's candidates (fp32 sums, as the definition has them)."""
    G, n, m = lp.shape
    out = [np.full((G, width), -1, np.int32), np.full((G, width), -1, np.int32),
           np.full((G, width), -np.inf, np.float32), np.ones((G, width), np.int32)]
    for g in range(G):
        cand = []
        for b in range(n):
            ended = done is not None and done[g, b] != 0
            for j in range(1 if ended else m):
                s = np.float32(scores[g, b]) if ended else np.float32(np.float32(scores[g, b]) + np.float32(lp[g, b, j]))
                if (ended or ids[g, b, j] >= 0) and s > -np.inf:
                    t = -1 if ended else int(ids[g, b, j])
                    cand.append((-float(s), b * m + j, g * n + b, t, s, int(ended or t in eos)))
        for r, c in enumerate(sorted(cand)[:width]):
            for o, v in zip(out, c[2:]):
                o[g, r] = v
    return out


def fork_ref(table, lens, parents, refs, free, at):
    """pages_fork step by step over Python lists: (table, lens, src, dst, status, refs, free)."""
    table, refs, free = np.array(table), [int(r) for r in refs], [int(f) for f in free]
    (S, W), N, P, F = table.shape, len(parents), len(refs), len(free)
    lens = [min(max(int(n), 0), W * PAGE) for n in lens]
    held = [-(-n // PAGE) for n in lens]
    old, at = list(refs), min(max(int(at), 0), F)
    new, nl = np.zeros((N, W), np.int64), [0] * N
    src, dst, refused, taken = [-1] * N, [-1] * N, 0, 0
    seen, first = set(), [False] * N
    for i, p in enumerate(parents):
        if 0 <= p < S and p not in seen:
            seen.add(p)
            first[i] = True
    keep = {}
    for i, p in enumerate(parents):
        p = int(p)
        if not 0 <= p < S:
            continue
        row, page = [int(v) for v in table[p, :held[p]]], -1
        if lens[p] % PAGE and 0 <= row[-1] < P and not (first[i] and old[row[-1]] == 1):
            page = free[at + taken] if at + taken < F else -1
            taken += 1
            if not 0 <= page < P:
                refused += 1
                continue
            src[i], dst[i], row[-1] = int(table[p, held[p] - 1]), page, page
        new[i, :held[p]], nl[i] = row, lens[p]
        for j in range(held[p]):
            if not (j == held[p] - 1 and page >= 0):
                keep[(p, j)] = keep.get((p, j), 0) + 1
    lost = set()
    for s in range(S):
        for j in range(held[s]):
            q, gain = int(table[s, j]), keep.get((s, j), 0) - 1
            if 0 <= q < P and gain:
                refs[q] += gain
                if gain < 0:
                    lost.add(q)
    here = at + min(taken, F - at)
    gone = sorted(q for q in lost if refs[q] == 0)
    back = max(here - len(gone), 0)
    for k, q in enumerate(gone[:here - back]):
        free[back + k] = q
    for d in dst:
        if d >= 0:
            refs[d] = 1
    status = [sum(d >= 0 for d in dst), back, refused, len(gone) - (here - back)]
    return new, nl, src, dst, status, refs, free
