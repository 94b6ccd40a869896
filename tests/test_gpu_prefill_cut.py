"""Prompt attention over the bf16 pool where a row block holds tokens on both sides of a key cut."""

from __future__ import annotations

import pytest
import torch

from jitengine_amd import ops

pytestmark = pytest.mark.gpu


def test_tokens_on_either_side_of_a_key_cut():
    """Blocks across the first key cut, more of them than the GPU runs at once: the items of the second part start
    after those of the first have ended, and leave the tokens before the cut as they are."""
    H, Hkv, ctx, n, many = 32, 4, 6130, 30, 90
    g = torch.Generator().manual_seed(12)
    npg = -(-(ctx + n) // 16)
    pool = torch.randn((npg, Hkv, 2, 16 * 128), generator=g).to(torch.bfloat16).cuda()
    table = torch.randperm(npg, generator=g).to(torch.int32).view(1, npg).cuda()
    q = torch.randn((n, H, 128), generator=g).to(torch.bfloat16).cuda()
    one = ops.paged_prefill_attention(q, pool, table, ops.prefill_plan([(0, ctx, n)], H, Hkv, "cuda"), 128 ** -0.5)
    plan = ops.prefill_plan([(0, ctx, n)] * many, H, Hkv, "cuda")
    out = ops.paged_prefill_attention(q.repeat(many, 1, 1), pool, table, plan, 128 ** -0.5)
    assert bool(torch.isfinite(out).all())
    assert torch.equal(out.view(torch.int16), one.repeat(many, 1, 1).view(torch.int16))
