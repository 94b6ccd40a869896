"""Scoring from hidden rows and the packed head: each of its kernels over long K and long runs of the head, running softmax
states that must follow the logits upwards, and rows whose sums overflow or lie far from 0."""

from __future__ import annotations

import pytest
import torch

from jitengine_amd import ops
from jitengine_amd.quant import random_quantized
from tests.test_gpu_scoring import DEV, U, _head, _head_ref

pytestmark = pytest.mark.gpu

# Tolerances of the softmax over logits that are exact, in half steps U of fp32.  A logit's exponential is off by ln 2 of
# its exponent's rounding, whose magnitude is below 72 + 16 (a reference lags by up to 64), and by 2 for the instruction; a
# join scales a state by another such exponential.  A wave folds up to 16 tiles, the 16 or 32 lanes of a row meet in 5
# additions, 8 waves in 8 joins, the runs in 4 + 6.
EXP = 0.7 * 88 + 2
JOINS = 18
REL = 16 + 5 + EXP + JOINS * (EXP + 2)  # of the sum of exponentials
OWN = 88 * (16 + 5 + 3 * JOINS)         # of the weighted sum alone, for roundings that it does not share with the other


def _softmax(z: torch.Tensor, tok: torch.Tensor):
    """(logprob, entropy, log of the sum, standard deviation of the logits under their distribution) of fp64 logits."""
    lse = torch.logsumexp(z, -1)
    p = torch.exp(z - lse[:, None])
    mean = (p * z).sum(-1)
    sd = torch.sqrt((p * (z - mean[:, None]) ** 2).sum(-1))
    return z.gather(1, tok.long()[:, None])[:, 0] - lse, torch.special.entr(p).sum(-1), lse, sd


def _check(r, lp, h, lse, sd, bound=0.0):
    """`bound`: how far the logits may be off."""
    tol = REL * U + 2 * bound
    assert torch.all((r.logprob.double() - lp).abs() <= tol + 1.25 * U * lp.abs())  # (log2 e is off by a quarter)
    assert torch.all((r.lse.double() - lse).abs() <= tol + 1.25 * U * lse.abs())
    # what both sums share moves the entropy by the logits' spread, the rest by the weighted sum's own roundings
    assert torch.all((r.entropy.double() - h).abs() <= (REL * U + bound) * (2 + 2 * sd) + OWN * U + U * h)
    assert float(r.logprob.max()) <= 0


def _tiles(T: int, K: int, V: int) -> int:
    """Token tiles of 32 that a workgroup of the kernel for many rows takes, from the workspace's size."""
    need, n32, found = ops.head_logprobs_workspace_bytes(T, K, V), (T + 31) // 32, set()
    for tt in range(1, 5):
        for tiles in range(-(-n32 // tt), -(-n32 // tt) + 1):
            t16 = 32 * tt * tiles
            g32 = (K // 64 + 31) // 32 * 32
            if need == (6 * t16 * g32 + 15) // 16 * 16 + 12 * 256 * (tiles // 256 + 2) * 32 * tt + 4 * T:
                assert tiles * (V // 16) // 256 >= 64  # (a run holds several walks of 32 blocks)
                found.add(tt)
    assert len(found) == 1
    return found.pop()


@pytest.mark.parametrize("T,V,tt,K", [(T, 151936, tt, K) for T, tt in ((130, 2), (282, 3), (300, 4), (512, 4))
                                      for K in (1920, 2048, 2176, 4224)] + [(24, 302000, 1, 4224)])
def test_many_rows_over_long_runs(T, V, tt, K):
    """Every tile of the kernel for many rows, over K below and above where the groups' sums fit LDS, with rows left over."""
    assert _tiles(T, K, V) == tt
    lin = _head(V, K, T + K)
    g = torch.Generator(device=DEV).manual_seed(T)
    x = (1.5 * torch.randn((T, K), generator=g, device=DEV)).to(torch.bfloat16)
    tok = torch.randint(0, V, (T,), generator=g, device=DEV, dtype=torch.int32)
    tok[:3] = torch.tensor([0, V - 1, V // 2])
    r = ops.head_logprobs(x, ops.prepack(lin), tok)
    lp, h, lse, bound = _head_ref(x, lin, tok)
    # (the spread: logits of standard deviation below 4 under any of these distributions)
    _check(r, lp, h, lse, 4.0, bound)


def _exact_head(target: torch.Tensor, K: int):
    """A head whose rows' logits against rows of a constant are exact: q of any value with scale 2^-8, biases that bring row v
    to about target[v] for a hidden row of ones (every term and sum is a multiple of 2^-10 below 2^9: fp32 loses nothing)."""
    V = target.numel()
    lin = random_quantized((V, K), 5, 0.02, DEV)
    lin.scales = torch.full_like(lin.scales, 2.0 ** -8)
    b = (target.double() / K - 7.5 / 256)[:, None].expand(V, K // 64)
    lin.biases = (torch.round(b * 2 ** 8) / 2 ** 8).to(torch.bfloat16).contiguous()
    q = (lin.weight.view(V, K // 8, 1) >> (4 * torch.arange(8, device=DEV, dtype=torch.int32))) & 15
    z = q.reshape(V, K).double().sum(-1) / 256 + 64 * lin.biases.double().sum(-1)
    return lin, z


def _along(kind: str, V: int, most: float) -> torch.Tensor:
    v = torch.arange(V, device=DEV) / V
    if kind == "rising":
        return most * v
    if kind == "falling":
        return most * (1 - v)
    if kind == "steps":  # a wave meets each part after the one before it
        return most * torch.floor(4 * v) / 4
    x = torch.zeros(V, device=DEV)
    x[-V // 50] = most  # one row near the end
    return x


@pytest.mark.parametrize("most", [20.0, 44.0, 60.0, 200.0])  # (a reference lags by up to 44.4)
@pytest.mark.parametrize("T", [1, 16, 50, 130, 300])
def test_states_follow_rising_logits(T, most):
    """Sums that a wave already holds when larger logits come, in each kernel: hidden rows of ones, halves and quarters give
    the same shape at three heights."""
    V, K = 400000, 256
    a = torch.tensor([1.0, 0.5, 0.25], device=DEV)[torch.arange(T, device=DEV) % 3]
    x = a[:, None].expand(T, K).to(torch.bfloat16).contiguous()
    g = torch.Generator(device=DEV).manual_seed(T)
    tok = torch.randint(0, V, (T,), generator=g, device=DEV, dtype=torch.int32)
    for kind in ("rising", "falling", "steps", "one"):
        lin, z = _exact_head(_along(kind, V, most), K)
        tok[::2] = int(z.argmax())
        r = ops.head_logprobs(x, ops.prepack(lin), tok)
        for c in (1.0, 0.5, 0.25):
            at = torch.nonzero(a == c)[:, 0]
            if at.numel():
                ref = _softmax((c * z).expand(at.numel(), V), tok[at])
                _check(ops.HeadLogprobs(r.logprob[at], r.entropy[at], r.lse[at]), *ref)


@pytest.mark.parametrize("T", [1, 16, 50, 130])
@pytest.mark.parametrize("value", [1e36, 1.1e37, 3e38])
def test_rows_whose_sums_overflow_are_nan(T, value):
    """Products are formed before the scale: sums that overflow on the way, or logits far past 2^28, make their row NaN and
    no other."""
    V, K = 5008, 256
    lin = _head(V, K, 3)
    lin.scales = lin.scales.abs()  # (positive and negative values overflow to one side each)
    head = ops.prepack(lin)
    g = torch.Generator(device=DEV).manual_seed(T)
    x = torch.randn((T, K), generator=g, device=DEV).to(torch.bfloat16)
    tok = torch.randint(0, V, (T,), generator=g, device=DEV, dtype=torch.int32)
    want = ops.head_logprobs(x, head, tok)
    for sign in (1, -1):
        bad = x.clone()
        bad[T // 2, 3] = sign * value
        r = ops.head_logprobs(bad, head, tok)
        keep = [i for i in range(T) if i != T // 2]
        for w, t in zip((want.logprob, want.entropy, want.lse), (r.logprob, r.entropy, r.lse)):
            assert torch.isnan(t[T // 2]) and torch.equal(t[keep], w[keep])


@pytest.mark.parametrize("T", [1, 16, 50, 130])
def test_logits_far_from_zero(T):
    """Rows whose largest logit lies past +-2^28 / log2 e are NaN; nearer ones, and rows whose other logits lie as far below as
    they like, are numbers."""
    V, K = 5008, 256
    g = torch.Generator(device=DEV).manual_seed(T)
    tok = torch.randint(0, V, (T,), generator=g, device=DEV, dtype=torch.int32)
    for top, rest, nan in ((1.5e8, 1.5e8, False), (-1.5e8, -1.5e8, False), (0.0, -1e37, False), (2e8, 0.0, True),
                           (-2e8, -2e8, True), (1e12, 1e12, True), (1e30, 0.0, True), (-1e30, -1e30, True)):
        lin = random_quantized((V, K), 5, 0.02, DEV)
        lin.scales = torch.zeros_like(lin.scales)
        b = torch.full((V, 1), rest / K, device=DEV)
        b[V // 3] = top / K
        lin.biases = b.expand(V, K // 64).to(torch.bfloat16).contiguous()
        x = torch.ones((T, K), dtype=torch.bfloat16, device=DEV)
        r = ops.head_logprobs(x, ops.prepack(lin), tok)
        if nan:
            assert all(torch.isnan(t).all() for t in (r.logprob, r.entropy, r.lse))
        else:  # (sums of 256 equal bf16 numbers: exact)
            z = K * lin.biases[:, 0].double()
            lp, h, lse, sd = _softmax(z.expand(T, V), tok)
            _check(r, lp, h, lse, sd)
