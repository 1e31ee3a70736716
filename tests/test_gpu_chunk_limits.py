"""The prompt-chunk operators at the limits of their documentation: contexts
of 2^25 slots and more, lengths and starts that cannot be, rows of outputs
that lie apart.  64-bit restatements and tolerances are those of
test_gpu_chunk.py."""
import numpy as np
import pytest
import torch

import chunk_ref as R

pytestmark = pytest.mark.gpu
U = 2.0 ** -8


def _same(a, b):
    return torch.equal(a.contiguous().view(torch.uint8), b.contiguous().view(torch.uint8))


@pytest.mark.parametrize("heads,ctx_len", [(64, (1 << 25) + 77), (48, (1 << 26) + 5)])
def test_scores_of_a_very_long_context(ctx, heads, ctx_len):
    """One token, all of its heads on one KV head, over a cache whose every
    page is the same block: a slot's weight depends on its place in the page
    alone, and all weights add up to the heads.  (A page's 16 weights against
    their 64-bit values, to 2^-11: 1e-4 for scores and exponentials, and for
    the log-sum-exp's fp32 sum 2^26 slots / 148 CTAs / 128 a tile = 3543
    additions of half a step, 2^-24, each: 2.2e-4.)"""
    from kyro_b200.verify import chunk_attention, kv_scores_add
    d, pages = 64, (ctx_len + 1 + 15) // 16
    g = torch.Generator(device=ctx.device).manual_seed(3)

    def normal(*shape):
        return torch.randn(shape, generator=g, device=ctx.device).bfloat16()

    k, v, q = normal(1, 1, 16, d), normal(1, 1, 16, d), normal(1, heads, d)
    table = torch.zeros(1, pages, dtype=torch.int64, device=ctx.device)
    starts = torch.tensor([0, 1], dtype=torch.int32, device=ctx.device)
    lens = torch.tensor([ctx_len], device=ctx.device)
    lse = torch.empty(1, heads, device=ctx.device)
    chunk_attention(ctx, q, k, v, starts, table, lens, lse=lse)
    scores = torch.zeros(1, 1, pages * 16, device=ctx.device)
    kv_scores_add(ctx, q, k, lse, starts, table, lens, scores)
    assert ctx.device_status() == 0
    x = torch.exp(q[0].double() @ k[0, 0].double().T * d ** -0.5)  # [heads, 16]
    held = torch.tensor([(ctx_len + 1 + 15 - i) // 16 for i in range(16)], device=ctx.device)
    want = (x / (x * held).sum(-1, keepdim=True)).sum(0)
    got = scores[0, 0, :ctx_len + 1]
    for i in range(16):
        assert ((got[i::16].double() - want[i]).abs() <= 2.0 ** -11 * want[i]).all(), i
    assert (scores[0, 0, ctx_len + 1:] == 0).all()
