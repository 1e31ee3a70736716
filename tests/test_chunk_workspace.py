"""The workspace argument of the chunk operators and of the eviction: what a
kernel cannot write to is refused before one is launched."""
from types import SimpleNamespace

import pytest
import torch

import chunk_ref as R


def _calls(ctx, x, scores):
    from kyro_b200.verify import chunk_attention, kv_evict, kv_scores_add
    i32 = dict(dtype=torch.int32, device=x.q.device)
    lse = torch.zeros(x.T, x.hq, device=x.q.device)
    return [
        lambda w: chunk_attention(ctx, x.q, x.k_cache, x.v_cache, x.chunk_starts, x.block_table,
                                  x.context_lens, workspace=w),
        lambda w: kv_scores_add(ctx, x.q, x.k_cache, lse, x.chunk_starts, x.block_table,
                                x.context_lens, scores, workspace=w),
        lambda w: kv_evict(ctx, 16, 1, 1, [scores], [x.k_cache], [x.v_cache], x.block_table,
                           x.context_lens, torch.zeros(x.nb, **i32), torch.zeros(1, **i32),
                           torch.ones(x.nb, **i32), 16, workspace=w)]


def _refused(call, dev):
    for bad, error in ((torch.zeros(1 << 26, dtype=torch.uint8, device=dev)[::2], ValueError),
                       (torch.zeros(1 << 26, dtype=torch.uint8, device="meta"), ValueError),
                       (bytearray(1 << 26), TypeError), (1 << 40, TypeError)):
        with pytest.raises(error, match="workspace"):
            call(bad)


@pytest.mark.parametrize("which", [0, 1, 2])
def test_workspace_refusals(which):
    dev = torch.device("cpu")
    x = R.Batch(dev, [2, 1], [20, 3], 4, 2, 64)
    _refused(_calls(SimpleNamespace(device=dev), x, torch.zeros(2, 2, 64))[which], dev)


@pytest.mark.gpu
@pytest.mark.parametrize("which", [0, 1, 2])
def test_workspace_on_the_gpu(ctx, which):
    from kyro_b200._lib import KYRO_ERR_WORKSPACE, KyroError
    x = R.Batch(ctx.device, [2, 1], [20, 3], 4, 2, 64)
    scores = torch.zeros(2, 2, 64, device=ctx.device)
    call = _calls(ctx, x, scores)[which]
    _refused(call, ctx.device)
    with pytest.raises(ValueError, match="workspace"):
        call(torch.zeros(1 << 26, dtype=torch.uint8))
    with pytest.raises(KyroError) as e:
        call(torch.zeros(8, dtype=torch.uint8, device=ctx.device))
    assert e.value.status == KYRO_ERR_WORKSPACE
    first = None
    for dtype in (torch.uint8, torch.int32, torch.float64):  # bytes are bytes
        scores.zero_()
        r = call(torch.empty(1 << 26, dtype=torch.uint8, device=ctx.device).view(dtype))
        first = r.clone() if first is None else first
        assert torch.equal(r, first)
    assert ctx.device_status() == 0
