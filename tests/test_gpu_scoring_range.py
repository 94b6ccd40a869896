"""Rows of logits far from 0 against 64-bit ones: masks of large negative numbers that leave nothing, and what lies beside them;
lists of very many pages."""

from __future__ import annotations

import math

import pytest
import torch

from jitengine_amd import ops
from tests.test_gpu_scoring import DEV, U, _check_rows

pytestmark = pytest.mark.gpu


def _far(kind: str, V: int, dtype) -> torch.Tensor:
    """Six rows; what is not said is a normal row's numbers."""
    g = torch.Generator().manual_seed(V)
    n = 3 * torch.randn((6, V), generator=g)
    on = torch.rand((6, V), generator=g) < 0.5
    if kind == "nothing":  # every token ruled out, by one number
        x = torch.tensor([-1e9, -1e10, -1e30, -2.3e38, 1e12, 3e38])[:, None].expand(6, V)
    elif kind == "masked twice":  # ... and some of them for good, or further
        x = torch.full((6, V), -1e30)
        x[:3][on[:3]] = -math.inf
        x[3:][on[3:]] = -2e38
    elif kind == "one":  # one number stands out
        x = n.clone()
        x[:, V // 3] = torch.tensor([1e9, 1e12, 1e30, -1e30, 3e38, 7e6])
        x[3:5, V // 2:] = -1e30
    elif kind == "late":  # the first numbers of a row come behind more masked values than a wave has lanes
        x = torch.full((6, V), -1e30)
        x[:, V // 2:] = torch.where(on, n, -1e30)[:, V // 2:]
        x[4:] += torch.tensor([[5e4], [3e6]])
    else:  # numbers about the place where the other form of the exponent begins, and a row that walks past it
        x = torch.round(16 * n) / 16 + torch.tensor([726817.0, 726810.0, -726817.0, 1e6, -3e6, 0.0])[:, None]
        x[5] = torch.linspace(0, 3e6, V)
    return x.to(dtype)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32], ids=["bf16", "fp32"])
@pytest.mark.parametrize("kind", ["nothing", "masked twice", "one", "late", "border"])
@pytest.mark.parametrize("V,slices", [(70, 1), (9000, 4), (151936, 64)])
def test_token_logprobs_of_rows_far_from_zero(V, slices, kind, dtype):
    x = _far(kind, V, dtype)
    tok = torch.tensor([0, V - 1, V // 2, V // 3, V, 1], dtype=torch.int32)
    _check_rows(x, tok, 9, ops.token_logprobs(x.to(DEV), tok.to(DEV), top=9), slices)
    many = x.repeat(200, 1)  # (one workgroup a row)
    r = ops.token_logprobs(many.to(DEV), tok.repeat(200).to(DEV), top=9)
    _check_rows(x, tok, 9, ops.TokenLogprobs(*(t[-6:] for t in (r.logprob, r.rank, r.entropy, r.top_ids, r.top_logprobs))))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32], ids=["bf16", "fp32"])
@pytest.mark.parametrize("V", [100, 40000])
def test_token_logprobs_are_never_above_zero(V, dtype):
    """Rows whose mask leaves one token, and rows in which one has nearly everything: probabilities of 1, rounded."""
    B = 300
    g = torch.Generator().manual_seed(V)
    x = torch.full((B, V), -math.inf)
    tok = torch.randint(0, V, (B,), generator=g, dtype=torch.int32)
    x[torch.arange(B), tok.long()] = torch.linspace(2, 100, B)
    x[B // 2:] = torch.where(torch.isinf(x[B // 2:]), torch.linspace(-30, -20, V), x[B // 2:])
    x = x.to(dtype)
    r = ops.token_logprobs(x.to(DEV), tok.to(DEV), top=2)
    assert float(r.logprob.max()) <= 0 and float(r.top_logprobs.max()) <= 0 and float(r.entropy.min()) >= 0
    # (the sums hold one number of note: its exponential, up to a few joins, and the logarithm's argument are rounded)
    assert float(r.logprob.min()) >= -64 * U
    assert torch.equal(r.rank, torch.zeros_like(r.rank)) and torch.equal(r.top_ids[:, 0], tok.to(DEV))


def test_copies_of_more_pages_than_a_launch_takes():
    """140,000 entries in 128 layers, nearly all of them -1: a launch has 2^24 workgroups at most."""
    g = torch.Generator(device=DEV).manual_seed(1)
    pools = [torch.randn((12, 1, 2, 2048), generator=g, device=DEV).to(torch.bfloat16) for _ in range(128)]
    want = [p.clone() for p in pools]
    src, dst = (torch.full((140000,), -1, dtype=torch.int32) for _ in range(2))
    for at, s, d in ((0, 0, 6), (131070, 1, 7), (131071, 2, 8), (139999, 3, 9)):
        src[at], dst[at] = s, d
        for w in want:
            w[d] = w[s]
    ops.kv_copy_pages_layers(ops.pool_layers(pools), src.to(DEV), dst.to(DEV))
    assert all(torch.equal(p, w) for p, w in zip(pools, want))
