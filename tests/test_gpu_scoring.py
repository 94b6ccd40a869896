"""The scoring and continuation operators on the GPU against plain 64-bit and whole-number implementations."""

from __future__ import annotations

import math

import numpy as np
import pytest
import torch

from jitengine_amd import _lib, ops
from jitengine_amd.quant import random_quantized
from tests.scoring_ref import beams_ref, fork_ref, rows_ref

pytestmark = pytest.mark.gpu
DEV = "cuda"
U = 2.0 ** -24  # half a step of fp32


def _i32(a):
    return torch.from_numpy(np.ascontiguousarray(np.asarray(a, np.int32))).to(DEV)


def _rows(kind: str, B: int, V: int, dtype, seed: int) -> torch.Tensor:
    g = torch.Generator().manual_seed(seed)
    x = torch.randn((B, V), generator=g) * 3
    low = torch.finfo(dtype).min
    if kind == "ties":
        x = torch.round(x)
    elif kind == "constant":
        x = torch.full((B, V), 1.5)
    elif kind == "ascending":
        x = torch.linspace(-20, 20, V).repeat(B, 1)
    elif kind == "descending":
        x = torch.linspace(20, -20, V).repeat(B, 1)
    elif kind == "masked":
        x[torch.rand((B, V), generator=g) < 0.97] = -math.inf
    elif kind == "lowest":  # the type's lowest value beside numbers, and in a row of nothing else
        x[torch.rand((B, V), generator=g) < 0.5] = low
        x[0] = low
    elif kind == "nothing":
        x[0] = -math.inf
        x[-1, 1:] = -math.inf
    elif kind == "loud":  # one token has nearly everything
        x[:, V // 2] = 60
    elif kind == "odd":  # NaN, infinities, both zeros
        x[0, V // 3] = math.nan
        x[-1, V // 2] = math.inf
        x[B // 2] = torch.where(torch.arange(V) % 2 == 0, 0.0, -0.0)
    return x.to(dtype)


def _check_rows(x, tokens, top, r, slices=1):
    """Tolerances: e^(x - m) is off by 2^-23 of the exponent |d| log2 e < 150 where it counts (d < -104 gives 0), each lane
    adds V / (256 slices) + 32 of them one after the other and the joins some 16, half a step each; the log-probability and
    the entropy are rounded once."""
    lp, rank, ent, ids, tlp = rows_ref(x, tokens, top)
    adds = x.shape[1] / 256 / slices + 32 + 16
    rel = (adds + 2 * 20 + 4) * U  # (of l: the terms that make up l lie within e^-20 of the largest, or add less than U)
    if tokens is not None:
        assert torch.equal(r.rank.cpu().long(), rank)
        torch.testing.assert_close(r.logprob.cpu().double(), lp, rtol=U, atol=rel, equal_nan=True)
    # t / l: both sums off by rel, and |t| / l < 20 + ln V
    torch.testing.assert_close(r.entropy.cpu().double(), ent, rtol=U, atol=rel * (2 * 20 + 2 * math.log(x.shape[1]) + 1),
                               equal_nan=True)
    if top:
        assert torch.equal(r.top_ids.cpu().long(), ids)
        torch.testing.assert_close(r.top_logprobs.cpu().double(), tlp, rtol=U, atol=rel, equal_nan=True)


KINDS = ["normal", "ties", "constant", "ascending", "descending", "masked", "lowest", "nothing", "loud", "odd"]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32], ids=["bf16", "fp32"])
@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("V", [64, 1001, 9000])
def test_token_logprobs_of_every_kind_of_row(V, kind, dtype):
    x = _rows(kind, 5, V, dtype, seed=V)
    tok = torch.tensor([0, V - 1, V // 2, -1, V], dtype=torch.int32)
    for top in (0, 1, 7, 64):
        _check_rows(x, tok, top, ops.token_logprobs(x.to(DEV), tok.to(DEV), top=top))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32], ids=["bf16", "fp32"])
@pytest.mark.parametrize("B,V", [(1, 1), (1, 2), (3, 7), (2, 8), (2, 9), (1, 2048), (1, 2049), (4, 4097), (1, 151936),
                                 (40, 70001), (3, 248320)])
def test_token_logprobs_of_every_size(B, V, dtype):
    x = _rows("normal", B, V, dtype, seed=B + V)
    g = torch.Generator().manual_seed(V)
    tok = torch.randint(0, V, (B,), generator=g, dtype=torch.int32)
    top = min(V, 20)
    _check_rows(x, tok, top, ops.token_logprobs(x.to(DEV), tok.to(DEV), top=top))


def test_token_logprobs_of_many_rows_take_one_workgroup_each():
    assert ops.token_logprobs_workspace_bytes(2500, 3001) == 0
    x = _rows("ties", 2500, 3001, torch.bfloat16, 4)
    tok = torch.arange(2500, dtype=torch.int32)
    _check_rows(x, tok, 5, ops.token_logprobs(x.to(DEV), tok.to(DEV), top=5))


@pytest.mark.parametrize("m", [1, 2, 5, 64])
@pytest.mark.parametrize("B,V", [(3, 300), (2, 20000)])
def test_token_logprobs_of_several_tokens_a_row(B, V, m):
    x = _rows("ties", B, V, torch.bfloat16, m)
    g = torch.Generator().manual_seed(m)
    tok = torch.randint(-2, V + 2, (B, m), generator=g, dtype=torch.int32)
    _check_rows(x, tok, 3, ops.token_logprobs(x.to(DEV), tok.to(DEV), top=3))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32], ids=["bf16", "fp32"])
@pytest.mark.parametrize("at", [1, 3, 8])
def test_token_logprobs_of_rows_at_a_stride(at, dtype):
    """Rows inside wider ones, at addresses that no vector load takes; what lies around them is not read."""
    V = 5003
    wide = torch.full((4, V + 21), math.nan, dtype=dtype)
    x = _rows("ties", 4, V, dtype, 9)
    wide[:, at:at + V] = x
    tok = torch.tensor([0, 17, V - 1, 4], dtype=torch.int32)
    _check_rows(x, tok, 9, ops.token_logprobs(wide.to(DEV)[:, at:at + V], tok.to(DEV), top=9))


@pytest.mark.parametrize("top", [1, 31, 32, 33, 63, 64])
@pytest.mark.parametrize("kind", ["normal", "ties", "constant", "ascending", "descending", "masked"])
def test_token_logprobs_of_every_number_of_alternatives(kind, top):
    """Of a row in as many slices as there are, and of rows of several steps a workgroup."""
    for B, V, slices in ((1, 200000, 32), (600, 20001, 1)):
        x = _rows(kind, 3 if B > 1 else 1, V, torch.bfloat16, top)
        tok = torch.randint(0, V, (x.shape[0],), generator=torch.Generator().manual_seed(top), dtype=torch.int32)
        n = B // x.shape[0]
        r = ops.token_logprobs(x.repeat(n, 1).to(DEV), tok.repeat(n).to(DEV), top)
        k = x.shape[0]
        _check_rows(x, tok, top, ops.TokenLogprobs(*(t[-k:] for t in (r.logprob, r.rank, r.entropy, r.top_ids, r.top_logprobs))), slices)
        if B > 1:  # (24 rows on, a row of any length begins at the same place in its 16 bytes: the same sums in the same order)
            assert torch.equal(r.top_ids[:k], r.top_ids[24:24 + k]) and torch.equal(r.logprob[:k], r.logprob[24:24 + k])


def test_token_logprobs_without_rows_tokens_or_alternatives():
    r = ops.token_logprobs(torch.zeros((0, 50), device=DEV), _i32([]), top=3)
    assert r.logprob.shape == (0,) and r.top_ids.shape == (0, 3)
    x = _rows("normal", 3, 500, torch.float32, 1)
    r = ops.token_logprobs(x.to(DEV))
    assert r.logprob is None and r.rank is None and r.top_ids is None
    _check_rows(x, None, 0, r)
    with pytest.raises(ValueError, match="top=501"):
        ops.token_logprobs(x.to(DEV), top=501)
    with pytest.raises(_lib.UnsupportedShape):
        ops.token_logprobs(x.to(DEV), top=65)
    with pytest.raises(ValueError, match="tokens must be"):
        ops.token_logprobs(x.to(DEV), _i32([1, 2]))
    with pytest.raises(ValueError, match="workspace"):
        ops.token_logprobs(torch.zeros((1, 90000), device=DEV), workspace=torch.empty(16, dtype=torch.uint8, device=DEV))


def test_token_logprobs_of_very_long_rows_and_of_very_many():
    x = _rows("normal", 2, 3000001, torch.float32, 3)
    tok = torch.tensor([[2999999, 0], [7, 3000000]], dtype=torch.int32)
    _check_rows(x, tok, 9, ops.token_logprobs(x.to(DEV), tok.to(DEV), 9), 64)
    x = _rows("normal", 70000, 33, torch.bfloat16, 4)
    tok = (torch.arange(70000) % 35 - 1).to(torch.int32)
    r = ops.token_logprobs(x.to(DEV), tok.to(DEV), 3)
    at = torch.tensor([0, 1, 34, 35, 2047, 2048, 65535, 65536, 69998, 69999])
    _check_rows(x[at], tok[at], 3, ops.TokenLogprobs(*(t[at.to(DEV)] for t in (r.logprob, r.rank, r.entropy, r.top_ids, r.top_logprobs))))


def test_token_logprobs_of_rows_whose_largest_grows_slowly():
    """References lag behind values that grow by less than a step's worth; one value then has everything."""
    V = 40000
    for top in (7.9, 8.1, 40.0):
        x = torch.stack([torch.linspace(0, top, V), torch.linspace(0, top, V).flip(0), torch.cat([torch.zeros(V - 1), torch.tensor([top])])])
        tok = torch.tensor([V - 1, 0, V - 1], dtype=torch.int32)
        for rows in (x, x.repeat(400, 1)):  # (split rows, and whole ones)
            r = ops.token_logprobs(rows.to(DEV), tok.repeat(rows.shape[0] // 3).to(DEV), 5)
            _check_rows(x, tok, 5, ops.TokenLogprobs(*(t[:3] for t in (r.logprob, r.rank, r.entropy, r.top_ids, r.top_logprobs))))


def test_token_logprobs_past_4_gib():
    """Row offsets past 32 bits: the last row of logits of 4.2 GiB."""
    B, V = 15000, 151936
    x = torch.zeros((B, V), dtype=torch.bfloat16, device=DEV)
    last = _rows("normal", 1, V, torch.bfloat16, 3)
    x[-1] = last[0].to(DEV)
    tok = torch.full((B,), 77, dtype=torch.int32)
    r = ops.token_logprobs(x, tok.to(DEV), top=4)
    one = ops.TokenLogprobs(r.logprob[-1:], r.rank[-1:], r.entropy[-1:], r.top_ids[-1:], r.top_logprobs[-1:])
    _check_rows(last, tok[-1:], 4, one)
    assert torch.all(r.rank[:-1] == 77) and torch.all(r.top_ids[:-1] == _i32([0, 1, 2, 3]))


# ----------------------------------------------------------------------------- the head
def _head(V, K, seed, loud=False):
    lin = random_quantized((V, K), seed, 0.02, DEV)
    if loud:  # scales and biases of any size and sign
        g = torch.Generator(device=DEV).manual_seed(seed)
        f = torch.exp(1.5 * torch.randn(lin.scales.shape, generator=g, device=DEV))
        lin.scales = (lin.scales.float() * f * torch.sign(f - 0.7)).to(torch.bfloat16)
        lin.biases = (lin.biases.float() * torch.exp(1.5 * torch.randn(lin.scales.shape, generator=g, device=DEV))).to(torch.bfloat16)
    return lin


def _head_ref(x, lin, tok):
    """(logprob, entropy, lse, bound of a logit's error) in fp64.  A logit sums products of at most |x| |s| 31 in fp32, 64 of
    them in a row and then the K / 64 groups (and |x| (|b| + 16 |s|) once a group): with independent roundings of half a step
    its error has a standard deviation below sqrt(64 + K / 64 + 8) U sqrt(sum of the squares); 8 of them are allowed."""
    V, K = lin.out_dims, lin.in_dims
    q = (lin.weight.view(V, K // 8, 1) >> (4 * torch.arange(8, device=DEV, dtype=torch.int32))) & 15
    s, b = (t.double().repeat_interleave(64, 1) for t in (lin.scales, lin.biases))
    w = q.reshape(V, K).double() * s + b
    xd = x.double()
    z = xd @ w.t()
    size = 31 * s.abs() + b.abs() + 16 * s.abs()
    bound = 8 * math.sqrt(64 + K / 64 + 8) * U * torch.sqrt((xd * xd) @ (size * size).t())
    lse = torch.logsumexp(z, -1)
    p = torch.exp(z - lse[:, None])
    in_ = (tok >= 0) & (tok < V)
    lp = z.gather(1, tok.long().clamp(0, V - 1)[:, None])[:, 0] - lse
    return torch.where(in_, lp, 0.0), torch.special.entr(p).sum(-1), lse, bound.amax(-1)


def _check_head(x, lin, tok):
    r = ops.head_logprobs(x, ops.prepack(lin), tok)
    lp, h, lse, bound = _head_ref(x, lin, tok)
    V = lin.out_dims
    rel = (V / 256 + 128) * U  # (of the sum of exponentials: as for rows of logits, see _check_rows)
    tol = 2 * bound + rel
    assert torch.all((r.logprob.double() - lp).abs() <= tol + U * lp.abs())
    assert torch.all((r.lse.double() - lse).abs() <= tol + U * lse.abs())
    # dH = -sum p (ln p + H) dz: at most the bound times the mean of |ln p + H|, itself below 2 H + 2
    assert torch.all((r.entropy.double() - h).abs() <= bound * (2 * h + 2) + rel * (2 * math.log(V) + 41) + U * h)


@pytest.mark.parametrize("T", [1, 2, 15, 16, 17, 31, 32, 33, 63, 64, 65, 77, 128, 129, 200, 257, 300])
def test_head_logprobs_of_every_row_count(T):
    V, K = 2064, 256
    lin = _head(V, K, 3)
    g = torch.Generator(device=DEV).manual_seed(T)
    x = (3 * torch.randn((T, K), generator=g, device=DEV)).to(torch.bfloat16)
    tok = torch.randint(0, V, (T,), generator=g, device=DEV, dtype=torch.int32)
    _check_head(x, lin, tok)


@pytest.mark.parametrize("V", [16, 48, 64, 80, 1024, 1040, 5008])
@pytest.mark.parametrize("K", [128, 384, 2048, 4096, 4224])
@pytest.mark.parametrize("T", [1, 40, 150])
def test_head_logprobs_of_every_head(T, K, V):
    lin = _head(V, K, V + K, loud=True)
    g = torch.Generator(device=DEV).manual_seed(T)
    x = torch.randn((T, K), generator=g, device=DEV).to(torch.bfloat16)
    tok = torch.randint(-2, V + 2, (T,), generator=g, device=DEV, dtype=torch.int32)
    tok[0] = V - 1
    _check_head(x, lin, tok)


@pytest.mark.parametrize("K", [1920, 2176, 4096])
@pytest.mark.parametrize("T", [17, 50, 77, 96])
def test_head_logprobs_of_one_tile_over_several_passes(T, K):
    g = torch.Generator(device=DEV).manual_seed(T + K)
    lin = _head(30000, K, T)
    tok = torch.randint(0, 30000, (T,), generator=g, device=DEV, dtype=torch.int32)
    _check_head((2 * torch.randn((T, K), generator=g, device=DEV)).to(torch.bfloat16), lin, tok)


@pytest.mark.parametrize("T,V", [(1000, 48), (5000, 528), (40000, 32), (40001, 272)])
def test_head_logprobs_of_many_rows_and_a_small_head(T, V):
    """More token tiles than workgroups, whose runs meet several of them."""
    g = torch.Generator(device=DEV).manual_seed(T)
    lin = _head(V, 256, V)
    tok = torch.randint(-1, V + 1, (T,), generator=g, device=DEV, dtype=torch.int32)
    _check_head((2 * torch.randn((T, 256), generator=g, device=DEV)).to(torch.bfloat16), lin, tok)


@pytest.mark.parametrize("T", [1, 20, 130])
def test_head_logprobs_over_a_vocabulary(T):
    V, K = 151936, 512
    lin = _head(V, K, 8)
    g = torch.Generator(device=DEV).manual_seed(T)
    x = (2 * torch.randn((T, K), generator=g, device=DEV)).to(torch.bfloat16)
    tok = torch.randint(0, V, (T,), generator=g, device=DEV, dtype=torch.int32)
    _check_head(x, lin, tok)


@pytest.mark.parametrize("T", [3, 70])
def test_head_logprobs_keeps_a_bad_row_to_itself(T):
    """A NaN or an infinity in one hidden row makes that row NaN, and no other."""
    V, K = 1024, 256
    lin = _head(V, K, 5)
    g = torch.Generator(device=DEV).manual_seed(T)
    x = torch.randn((T, K), generator=g, device=DEV).to(torch.bfloat16)
    tok = torch.randint(0, V, (T,), generator=g, device=DEV, dtype=torch.int32)
    head = ops.prepack(lin)
    want = ops.head_logprobs(x, head, tok)
    bad = x.clone()
    bad[1, 7], bad[2, 200] = math.nan, math.inf
    got = ops.head_logprobs(bad, head, tok)
    for w, r in zip((want.logprob, want.entropy, want.lse), (got.logprob, got.entropy, got.lse)):
        assert torch.isnan(r[1:3]).all()
        keep = [i for i in range(T) if i not in (1, 2)]
        assert torch.equal(r[keep], w[keep])


def test_head_logprobs_refusals():
    lin = _head(64, 256, 1)
    head, x = ops.prepack(lin), torch.zeros((2, 256), dtype=torch.bfloat16, device=DEV)
    with pytest.raises(ValueError, match="head_logprobs takes"):
        ops.head_logprobs(x[:, :128].contiguous(), head, _i32([0, 1]))
    with pytest.raises(ValueError, match="head_logprobs takes"):
        ops.head_logprobs(x, head, _i32([0]))
    with pytest.raises(_lib.UnsupportedShape):
        ops.head_logprobs(x, lin, _i32([0, 1]))
    with pytest.raises(ValueError, match="workspace"):
        ops.head_logprobs(x, head, _i32([0, 1]), torch.empty(8, dtype=torch.uint8, device=DEV))
    assert ops.head_logprobs(x[:0], head, _i32([])).logprob.shape == (0,)


# ----------------------------------------------------------------------------- beams
@pytest.mark.parametrize("G,n,m,w", [(1, 1, 1, 1), (1, 4, 8, 4), (3, 5, 7, 9), (2, 16, 16, 16), (5, 16, 33, 16), (2, 64, 64, 64),
                                     (1, 2, 3, 64), (70, 8, 16, 8)])
@pytest.mark.parametrize("kind", ["normal", "ties", "few"])
def test_beam_select(G, n, m, w, kind):
    rng = np.random.default_rng(G * n + m)
    scores, lp = rng.normal(-20, 5, (G, n)).astype(np.float32), -rng.exponential(2, (G, n, m)).astype(np.float32)
    ids = rng.integers(0, 50, (G, n, m)).astype(np.int32)
    done = (rng.random((G, n)) < 0.25).astype(np.int32) * 3
    if kind == "ties":
        scores, lp = np.round(scores / 4), np.round(lp)
    elif kind == "few":
        lp[rng.random(lp.shape) < 0.8] = -np.inf
        ids[rng.random(ids.shape) < 0.5] = -1
        scores[rng.random(scores.shape) < 0.2] = -np.inf
        scores[rng.random(scores.shape) < 0.1] = np.nan
        lp[rng.random(lp.shape) < 0.1] = np.nan
    eos = (3, 17)
    for d, e in ((None, ()), (done, eos)):
        want = beams_ref(scores, lp, ids, w, d, e)
        r = ops.beam_select(torch.from_numpy(scores).to(DEV), torch.from_numpy(lp).to(DEV), _i32(ids), width=w,
                            done=None if d is None else _i32(d), eos=_i32(e) if e else None)
        for got, ref in zip((r.parents, r.tokens, r.scores, r.done), want):
            assert np.array_equal(got.cpu().numpy(), ref)


def test_beam_select_takes_the_best_token_of_logits_too():
    """top alternatives of token_logprobs straight into beam_select: the step of a beam search."""
    G, n, V = 2, 3, 4001
    x = _rows("normal", G * n, V, torch.bfloat16, 2)
    r = ops.token_logprobs(x.to(DEV), top=2 * n)
    s = torch.zeros((G, n), device=DEV)
    b = ops.beam_select(s, r.top_logprobs.view(G, n, -1), r.top_ids.view(G, n, -1))
    lp = torch.log_softmax(x.double(), -1).view(G, n * V)
    best = lp.sort(dim=-1, descending=True).values
    assert torch.allclose(b.scores.cpu().double(), best[:, :n], atol=1e-5)
    assert b.parents.shape == (G, n) and b.done.sum() == 0


# ----------------------------------------------------------------------------- pages
def _sequences(rng, S, W, P, shared):
    """Tables of S sequences over a pool of P pages, the first `shared` pages of each group of four in common."""
    perm, at = rng.permutation(P), 0
    table, lens = np.zeros((S, W), np.int64), rng.integers(0, W * 16 + 1, S)
    for s in range(S):
        held = -(-int(lens[s]) // 16)
        k = min(shared, held, int(lens[s]) // 16, -(-int(lens[s - 1]) // 16)) if s % 4 else 0
        table[s, :k] = table[s - 1, :k]
        table[s, k:held] = perm[at:at + held - k]
        at += held - k
    refs = np.zeros(P, np.int64)
    for s in range(S):
        refs[table[s, :-(-int(lens[s]) // 16)]] += 1
    return table, lens, refs, perm, at


def _fork_both(table, lens, parents, refs, free, at):
    want = fork_ref(table, lens, parents, refs, free, at)
    r_, f_ = _i32(refs), _i32(free)
    r = ops.pages_fork(_i32(table), _i32(lens), _i32(parents), r_, f_, _i32([at]))
    for got, ref in zip((r.page_table, r.lens, r.src, r.dst, r.status, r_, f_), want):
        assert np.array_equal(got.cpu().numpy(), np.asarray(ref).reshape(got.shape)), (got, ref)
    return r, r_, f_


@pytest.mark.parametrize("S,N,W,shared", [(1, 1, 1, 0), (1, 8, 3, 0), (4, 4, 20, 9), (8, 3, 300, 200), (33, 70, 17, 5),
                                          (1, 0, 4, 0), (300, 257, 9, 4), (1100, 1100, 3, 1)])
def test_pages_fork(S, N, W, shared):
    for seed in range(4):
        rng = np.random.default_rng(100 * S + seed)
        P = S * W + N + 5
        table, lens, refs, perm, at = _sequences(rng, S, W, P, shared)
        parents = rng.integers(-1, S + (seed == 1), N)
        if seed == 2:
            refs[table[:, 0]] += 1  # the first page has a holder outside
        if seed == 3:
            P_free = perm[:at + max(0, N // 4)]  # a list that ends too early
        else:
            P_free = perm
        _fork_both(table, lens, parents, refs, P_free, at)


def test_pages_fork_of_tables_with_ids_outside_the_pool():
    table = np.array([[5, 99, 2], [5, -7, 3]])
    _fork_both(table, [40, 26], [0, 1, 1, 0], np.array([0, 0, 1, 1, 0, 2, 0]), np.array([5, 2, 3, 0, -4, 6, 1]), 3)
    # lengths past the table hold what it has, negative ones nothing
    _fork_both(table, [1000, -3], [0, 0, 1], np.array([0, 0, 1, 1, 0, 2, 0]), np.array([5, 2, 3, 0, 4, 6, 1]), 3)


def test_pages_fork_where_the_list_has_no_room():
    """Pages that come back before the list's beginning are counted, and the lowest ones kept."""
    r, _, free = _fork_both(np.array([[1, 2], [3, 4]]), [32, 32], [-1], np.array([0, 1, 1, 1, 1]), np.array([9, 9, 0]), 2)
    assert r.status.tolist() == [0, 0, 0, 2] and free.tolist() == [1, 2, 0]


def test_pages_fork_of_large_tables():
    rng = np.random.default_rng(5)
    table, lens, refs, perm, at = _sequences(rng, 64, 2100, 64 * 2100 + 70, 1500)
    _fork_both(table, lens, rng.integers(0, 64, 64), refs, perm, at)


def test_forks_and_steps_keep_the_books():
    """Forks and step tables in turn on the device: after each, every page is held as often as its count says, and the
    list has exactly the pages that nobody holds."""
    rng = np.random.default_rng(11)
    P, W, S = 400, 40, 6
    refs, free, at = torch.zeros(P, dtype=torch.int32, device=DEV), _i32(rng.permutation(P)), _i32([0])
    table, lens = torch.zeros((S, W), dtype=torch.int32, device=DEV), _i32([0] * S)
    for turn in range(12):
        new = _i32(rng.integers(0, 30, table.shape[0]))
        t = ops.step_tables(lens, new, table, 1000, free=free, free_at=at)
        assert int(t.status[2]) == 0
        grown = free[int(at):int(t.status[1])].long()
        refs[grown] += 1
        r = ops.pages_fork(table, t.lens, _i32(rng.integers(-1, table.shape[0], S)), refs, free, t.status[1:2])
        assert int(r.status[2]) == int(r.status[3]) == 0
        table, lens, at = r.page_table, r.lens, r.status[1:2].clone()
        count = np.zeros(P, np.int64)
        for row, n in zip(table.cpu().numpy(), lens.cpu().numpy()):
            np.add.at(count, row[:-(-int(n) // 16)], 1)
        assert np.array_equal(refs.cpu().numpy(), count)
        assert np.array_equal(np.sort(free.cpu().numpy()[int(at):]), np.nonzero(count == 0)[0])


@pytest.mark.parametrize("kv8", [False, True])
@pytest.mark.parametrize("layers,P,Hkv,n", [(1, 5, 1, 2), (3, 40, 4, 17), (130, 6, 2, 3), (48, 64, 3, 30)])
def test_copy_pages_in_every_layer(layers, P, Hkv, n, kv8):
    g = torch.Generator(device=DEV).manual_seed(layers)
    pools = []
    for _ in range(layers):
        if kv8:
            pools.append(torch.randint(0, 256, (P, Hkv, ops.KV8_RECORD), generator=g, device=DEV, dtype=torch.uint8))
        else:
            pools.append(torch.randn((P, Hkv, 2, 2048), generator=g, device=DEV).to(torch.bfloat16))
    rng = np.random.default_rng(n)
    perm = rng.permutation(P)
    src, dst = perm[rng.integers(0, P - n, n)], perm[P - n:].copy()  # (a page may be copied several times)
    dst[n // 2] = -1
    want = []
    for p in pools:
        w = p.clone()
        for s, d in zip(src, dst):
            if d >= 0:
                w[d] = p[s]
        want.append(w)
    ops.kv_copy_pages_layers(ops.pool_layers(pools), _i32(src), _i32(dst))
    for p, w in zip(pools, want):
        assert torch.equal(p.view(torch.uint8), w.view(torch.uint8))


def test_copy_pages_refusals():
    a, b = (torch.zeros((4, 1, 2, 2048), dtype=torch.bfloat16, device=DEV) for _ in range(2))
    with pytest.raises(ValueError, match="twice"):
        ops.pool_layers([a, a])
    with pytest.raises(ValueError, match="pool 1 is"):
        ops.pool_layers([a, b[:3]])
    with pytest.raises(ValueError, match="must be torch.bfloat16"):
        ops.pool_layers([a, ops.kv8_pool(4, 1, DEV)])
    layers = ops.pool_layers([a, b])
    with pytest.raises(ValueError, match="equal-length"):
        ops.kv_copy_pages_layers(layers, _i32([0]), _i32([1, 2]))
    a[0] = 7
    ops.kv_copy_pages_layers(layers, _i32([0, 0, 9, -1]), _i32([4, -1, 1, 2]))  # (ids outside the pool copy nothing)
    assert float(a[1:].abs().max()) == 0


# ----------------------------------------------------------------------------- streams and graphs
def test_a_step_on_another_stream_and_in_a_graph():
    """Scoring, choice, fork and copy as one captured step, replayed over new contents: each replay is the eager result."""
    G, n, V, K, P, W = 2, 4, 2064, 256, 64, 6
    lin = _head(V, K, 1)
    head = ops.prepack(lin)
    g = torch.Generator(device=DEV).manual_seed(1)
    pools = [torch.randn((P, 1, 2, 2048), generator=g, device=DEV).to(torch.bfloat16) for _ in range(3)]
    layers = ops.pool_layers(pools)
    x = torch.empty((G * n, K), dtype=torch.bfloat16, device=DEV)
    tok, sc = torch.empty(G * n, dtype=torch.int32, device=DEV), torch.zeros((G, n), device=DEV)
    rng = np.random.default_rng(2)
    table, lens, refs0, perm, at = _sequences(rng, G * n, W, P, 2)
    table, lens, free0, at = _i32(table), _i32(lens), _i32(perm), _i32([at])
    refs0 = _i32(refs0)
    refs, free = refs0.clone(), free0.clone()

    def step():
        h = ops.head_logprobs(x, head, tok)
        r = ops.token_logprobs(ops.qmm(x, head), tok, top=8)
        b = ops.beam_select(sc, r.top_logprobs.view(G, n, -1), r.top_ids.view(G, n, -1))
        f = ops.pages_fork(table, lens, b.parents.view(-1), refs, free, at)
        ops.kv_copy_pages_layers(layers, f.src, f.dst)
        return [h.logprob, h.entropy, h.lse, r.logprob, r.rank, r.entropy, r.top_ids, r.top_logprobs, b.parents, b.tokens,
                b.scores, b.done, f.page_table, f.lens, f.src, f.dst, f.status]

    def fresh(seed):
        gg = torch.Generator(device=DEV).manual_seed(seed)
        x.copy_(3 * torch.randn(x.shape, generator=gg, device=DEV))
        tok.copy_(torch.randint(0, V, tok.shape, generator=gg, device=DEV))
        refs.copy_(refs0)
        free.copy_(free0)
        for i, p in enumerate(pools):
            p.copy_(torch.randn(p.shape, generator=gg, device=DEV) + i)

    side = torch.cuda.Stream()
    fresh(0)
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()  # (warm)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    for seed in range(1, 5):
        fresh(seed)
        want = [t.clone() for t in step()] + [refs.clone(), free.clone()] + [p.clone() for p in pools]
        fresh(seed)
        graph.replay()
        torch.cuda.synchronize()
        for w, t in zip(want, out + [refs, free] + pools):
            assert torch.equal(w.view(torch.uint8), t.view(torch.uint8))
        fresh(seed)
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            got = step()
        torch.cuda.current_stream().wait_stream(side)
        for w, t in zip(want, got):
            assert torch.equal(w.view(torch.uint8), t.view(torch.uint8))
