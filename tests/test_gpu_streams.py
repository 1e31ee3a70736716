"""Calls go to torch's current stream, whatever stream the context had."""
import ctypes as C

import numpy as np
import pytest
import torch

import chunk_ref as R

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("module", [True, False])
def test_a_stream_set_through_the_handle_is_bound_anew(monkeypatch, module):
    """The caller gives the context a busy stream through the public handle; the
    next call is the current stream's all the same, and done when that is."""
    from kyro_b200 import _lib
    from kyro_b200.verify import Context, kv_write, qk_norm_rope_kv_write
    if not torch.cuda.is_available():
        pytest.skip("no CUDA device")
    if not module:
        monkeypatch.setattr(_lib, "calls", lambda: None)
    ctx = Context(0)
    x = R.Batch(ctx.device, [4, 4], [20, 20], 4, 2, 64, seed=1)

    def new():
        return qk_norm_rope_kv_write(ctx, x.q, x.k_new, x.v_new, x.chunk_starts, x.block_table,
                                     x.context_lens, x.k_cache, x.v_cache, 16)

    def old():
        kv_write(ctx, x.k_new.view(2, 4, 2, 64), x.v_new.view(2, 4, 2, 64), x.block_table,
                 x.context_lens, x.k_cache, x.v_cache, 16)
        return x.v_cache

    for call in (new, old):
        want = call().clone()
        torch.cuda.synchronize()
        side = torch.cuda.Stream()
        x.v_cache.zero_()
        torch.cuda.synchronize()
        with torch.cuda.stream(side):
            torch.cuda._sleep(400_000_000)  # 0.2 s
        assert _lib.load().kyro_ctx_set_stream(ctx.handle, C.c_void_p(side.cuda_stream)) == 0
        got = call().clone()
        torch.cuda.current_stream().synchronize()
        assert not side.query()
        if call is old:  # (the values that the call stores, nothing else in the cache)
            for b in range(2):
                blk, off = x.where(b, np.arange(20, 24))
                assert torch.equal(got[blk, :, off], want[blk, :, off])
        else:
            assert torch.equal(got, want)
        side.synchronize()
    assert ctx.device_status() == 0


def test_a_closed_context_refuses(ctx):  # (ctx: there is a GPU)
    from kyro_b200._lib import KyroError
    from kyro_b200.verify import Context
    c = Context(0)
    c.close()
    with pytest.raises(KyroError, match="kyro_ctx"):
        c.bind_stream()
