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


def _bad_starts(kind, B, n):
    rng = np.random.default_rng(7)
    s = np.arange(B + 1) * n
    if kind == "scattered":  # a few entries that go back into the sequence before
        s[np.arange(2, B - 8, 9) + rng.integers(0, 7)] -= n + 1
    elif kind == "reversed":
        s = s[::-1].copy()
    elif kind == "past the end":
        s[-1] += 1
    elif kind == "below zero":
        s[0] = -1
    elif kind == "starts late":
        s[0] = s[1] + 1
    return [int(i) for i in s]


@pytest.mark.parametrize("starts", [[0, 4, -1, 12], [0, 12, 13, 13], [0, 4, 3, 12], [0, 4, 8, 13],
                                    [-1, 4, 8, 12], [5, 4, 8, 12], [0, 8, 4, 12], [12, 8, 4, 0],
                                    [0, 0, 12, 12], [0, 4, 13, 12]] +
                         [_bad_starts(k, 100, 3) for k in (
                             "scattered", "reversed", "past the end", "below zero",
                             "starts late")] + [_bad_starts("scattered", 1500, 2)])
def test_norm_rope_write_beside_bad_starts(ctx, starts):
    """Sequences whose starts cannot be are flagged and left out, the others
    served, whatever order the starts are in."""
    from kyro_b200._lib import DEV_BAD_LENGTH
    from kyro_b200.verify import qk_norm_rope_kv_write
    B = len(starts) - 1
    T = 12 if B == 3 else B * (3 if B == 100 else 2)
    lens = [20 + b % 5 for b in range(B)]
    # (each sequence has room for all rows)
    x = R.Batch(ctx.device, [12] * B, lens, 2, 1, 64, seed=1)
    q, k, v = (torch.randn(T, h, 64, device=ctx.device).bfloat16() for h in (2, 1, 1))
    out, kc, vc = torch.full_like(q, 7.0), x.k_cache.clone(), x.v_cache.clone()
    st = torch.tensor(starts, dtype=torch.int32, device=ctx.device)
    qk_norm_rope_kv_write(ctx, q, k, v, st, x.block_table, x.context_lens, kc, vc, 16, q_out=out)
    width = x.block_table.shape[1] * 16
    good = [b for b in range(B) if 0 <= starts[b] <= starts[b + 1] <= T
            and (starts[b] == starts[b + 1] or lens[b] + starts[b + 1] - starts[b] <= width)]
    assert ctx.device_status() == (0 if len(good) == B else DEV_BAD_LENGTH)
    for t in range(T):
        held = [b for b in good if starts[b] <= t < starts[b + 1]]
        if not held:
            assert (out[t] == 7.0).all()
            continue
        fits = 0
        for b in held:
            slot = lens[b] + t - starts[b]
            at = torch.tensor([slot], device=ctx.device)
            ref, mag = R.norm_rope(q[t:t + 1], None, at, 0.0, 10000.0)
            rk, mk = R.norm_rope(k[t:t + 1], None, at, 0.0, 10000.0)
            blk, off = int(x.host_table[b, slot // 16]), slot % 16
            fits += int(((out[t].double() - ref[0]).abs()
                         <= U * ref[0].abs() + 2.0 ** -20 * mag[0]).all() and
                        ((kc[blk, :, off].double() - rk[0]).abs()
                         <= U * rk[0].abs() + 2.0 ** -20 * mk[0]).all() and
                        _same(vc[blk, :, off], v[t]))
        assert fits >= 1, (t, held)


@pytest.mark.parametrize("length", [(1 << 63) - 1, (1 << 63) - 4, 1 << 62, (1 << 32) + 20, 1 << 31,
                                    -1, -(1 << 31) + 20, -(1 << 63)])
def test_lengths_that_no_table_holds(ctx, length):
    """Flagged and left out, however the new rows are added to them."""
    from kyro_b200._lib import DEV_BAD_LENGTH
    from kyro_b200.verify import chunk_attention, kv_evict, kv_scores_add, qk_norm_rope_kv_write
    x = R.Batch(ctx.device, [4, 4, 4], [20, 20, 20], 4, 2, 64, seed=1)
    want, lse = torch.empty_like(x.q), torch.zeros(x.T, x.hq, device=ctx.device)
    chunk_attention(ctx, x.q, x.k_cache, x.v_cache, x.chunk_starts, x.block_table, x.context_lens,
                    out=want, lse=lse)
    lens = x.context_lens.clone()
    lens[1] = length
    out, ls = torch.full_like(x.q, 7.0), torch.full_like(lse, 7.0)
    chunk_attention(ctx, x.q, x.k_cache, x.v_cache, x.chunk_starts, x.block_table, lens, out=out,
                    lse=ls)
    assert ctx.device_status() == DEV_BAD_LENGTH
    assert (out[4:8] == 7.0).all() and (ls[4:8] == 7.0).all()
    assert _same(out[:4], want[:4]) and _same(out[8:], want[8:])
    s = torch.full((3, 2, 200), 3.0, device=ctx.device)
    kv_scores_add(ctx, x.q, x.k_cache, lse, x.chunk_starts, x.block_table, lens, s)
    assert ctx.device_status() == DEV_BAD_LENGTH
    assert (s[1] == 3.0).all() and (s[0, :, :20] > 3.0).all() and (s[2, :, :20] > 3.0).all()
    kc, vc = x.k_cache.clone(), x.v_cache.clone()
    qk_norm_rope_kv_write(ctx, x.q, x.k_new, x.v_new, x.chunk_starts, x.block_table, lens, kc, vc,
                          16, q_out=out.fill_(7.0))
    assert ctx.device_status() == DEV_BAD_LENGTH and (out[4:8] == 7.0).all()
    blk, off = x.where(1, np.arange(24))
    assert _same(kc[blk, :, off], x.k_cache[blk, :, off])
    assert not (out[:4] == 7.0).all() and not (out[8:] == 7.0).all()
    free = torch.arange(x.nb, dtype=torch.int32, device=ctx.device)
    refs = torch.ones(x.nb, dtype=torch.int32, device=ctx.device)
    kept = torch.empty(1, 3, 2, 8, dtype=torch.int32, device=ctx.device)
    table, top = x.block_table.clone(), torch.zeros(1, dtype=torch.int32, device=ctx.device)
    gone = kv_evict(ctx, 8, 1, 2, [s], [kc], [vc], table, lens, free, top, refs, 16,
                    num_reserved=5, kept=kept)
    assert gone.tolist() == [-1, -1 if length > 8 else 0, -1]  # (no free blocks)
    assert ctx.device_status() == (DEV_BAD_LENGTH if length > 8 else 0)
    assert torch.equal(table, x.block_table) and int(lens[1]) == length and (kept == -1).all()


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("base,gap", [(0, 8), (0, 16), (8, 16), (8, 24), (16, 48)])
@pytest.mark.parametrize("chunks,ctxs", [([300, 1, 70], [0, 40, 17]), ([3], [9000]),
                                         ([1] * 30, list(range(0, 30 * 90, 90)))])
def test_attention_into_rows_that_lie_apart(ctx, d, base, gap, chunks, ctxs):
    """An output that is part of wider rows, on 16 and on 32 bytes, from whole
    items and from joined ones: the same bits as a dense one, and nothing
    beside them."""
    from kyro_b200.verify import chunk_attention
    x = R.Batch(ctx.device, chunks, ctxs, 8, 2, d, seed=d + gap, front=2, back=1)
    row = x.hq * d

    def call(out):
        lse = torch.full((x.T, x.hq), 7.0, device=ctx.device)
        chunk_attention(ctx, x.q, x.k_cache, x.v_cache, x.chunk_starts, x.block_table,
                        x.context_lens, out=out, lse=lse)
        return lse

    want = torch.full((x.T, x.hq, d), 7.0, dtype=torch.bfloat16, device=ctx.device)
    want_lse = call(want)
    ref, _, mag = R.attention(x)
    err = (want.double() - ref).abs()[2:-1]
    assert (err <= (U * ref.abs() + (U + 2.0 ** -11) * mag)[2:-1]).all()
    whole = torch.full((x.T, row + gap), 7.0, dtype=torch.bfloat16, device=ctx.device)
    # (a view that begins `base` elements into its rows)
    out = whole[:, base:base + row].unflatten(1, (x.hq, d))
    lse = call(out)
    assert ctx.device_status() == 0
    assert _same(out, want) and _same(lse, want_lse)
    assert (whole[:, :base] == 7.0).all() and (whole[:, base + row:] == 7.0).all()


@pytest.mark.parametrize("gap", [8, 32])
def test_norm_rope_into_rows_that_lie_apart(ctx, gap):
    from kyro_b200.verify import qk_norm_rope_kv_write
    x = R.Batch(ctx.device, [70, 1, 9], [3, 40, 0], 6, 2, 128, seed=gap, gap=gap, front=1, back=2)
    args = (x.k_new, x.v_new, x.chunk_starts, x.block_table, x.context_lens, x.k_cache, x.v_cache,
            16)
    want = qk_norm_rope_kv_write(ctx, x.q, *args, q_out=torch.full(
        (x.T, 6, 128), 7.0, dtype=torch.bfloat16, device=ctx.device))
    whole = torch.full((x.T, 6 * 128 + gap), 7.0, dtype=torch.bfloat16, device=ctx.device)
    out = whole[:, 8:8 + 6 * 128].unflatten(1, (6, 128))
    qk_norm_rope_kv_write(ctx, x.q, *args, q_out=out)
    assert ctx.device_status() == 0 and _same(out, want)
    assert (whole[:, :8] == 7.0).all() and (whole[:, 8 + 6 * 128:] == 7.0).all()


@pytest.mark.parametrize("width,sequences", [(32768, 60), (49152 - 64, 20), (131072, 30)])
def test_evict_short_rows_of_a_wide_table(ctx, width, sequences):
    """Tables far wider than their sequences, as a server's are, and many
    sequences: selections that hold their rows on chip and ones that do not."""
    import test_gpu_evict as E
    lens = [(37 * i) % 700 + 1 for i in range(sequences)]
    st, s, k, v = E._state(ctx.device, lens, 2, 8, 1, 16, 211, 3, seed=sequences,
                           width_extra=width // 16)
    ev, flags = E._run(ctx, st, s, k, v, 211, 3, 50, 3, 16)
    assert flags == 0 and all((e > 0) == (n > 211) for e, n in zip(ev, lens))


@pytest.mark.parametrize("odd", [-(1 << 31), -(1 << 31) + 5, (1 << 31) - 1])
def test_norm_rope_write_beside_starts_of_any_size(ctx, odd):
    """A start at the ends of its type, behind the sequence that holds the rows."""
    from kyro_b200._lib import DEV_BAD_LENGTH
    from kyro_b200.verify import qk_norm_rope_kv_write
    x = R.Batch(ctx.device, [8, 8, 8], [20, 20, 20], 2, 1, 64, seed=1)
    args = (x.block_table, x.context_lens, x.k_cache, x.v_cache, 16)
    q, k, v = x.q[:12], x.k_new[:12], x.v_new[:12]

    def call(starts):
        out = torch.full_like(q, 7.0)
        qk_norm_rope_kv_write(ctx, q, k, v, torch.tensor(starts, dtype=torch.int32,
                                                         device=ctx.device), *args, q_out=out)
        return out, ctx.device_status()

    want, flags = call([0, 8, 8, 8])
    assert flags == 0 and not (want[:8] == 7.0).all(-1).any()
    got, flags = call([0, 8, odd, 12])
    assert flags == DEV_BAD_LENGTH
    assert _same(got[:8], want[:8]) and (got[8:] == 7.0).all()
