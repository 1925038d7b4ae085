"""Single tokens whose keys are NaN over a whole part of the softmax (a warp's tiles, a run of keys): the result is NaN, whatever the
other parts hold."""
import pytest
import torch

from prefix_util import check_close, definition, make_batch
from mdma_b200 import ops, ops_tensor

DEV = "cuda"
OWN = [(0, [(1500, 1)]), (0, [(40, 1)]), (0, [(700, 1)]), (0, [(900, 1)])]


def spoiled(heads, kv_heads, dim, page_size, lo, hi):
    ctx, q, view, dense = make_batch(OWN, heads, kv_heads, dim, page_size, torch.bfloat16, 8, DEV)
    bad = max(range(4), key=lambda i: dense[i][0].shape[0])              # the longest
    at = torch.arange(lo, min(hi, dense[bad][0].shape[0]))
    pages = view.page_table[int(ctx.seq_slot[bad])].cpu().long()[at // page_size]
    view.k[pages.to(DEV), (at % page_size).to(DEV)] = float("nan")
    dense[bad][0][at] = float("nan")
    return ctx, q, view, dense, bad


def compare(out, ctx, q, dense, bad, heads, kv_heads, dim):
    want, size, spread, keys = definition(ctx, q, dense, heads, kv_heads, dim, dim ** -0.5)
    keep = torch.tensor([i != bad for i in range(4)])
    assert torch.isnan(want[bad]).all() and torch.isnan(out[bad]).all(), f"{int(torch.isfinite(out[bad]).sum())} finite numbers"
    check_close(out.cpu()[keep], (want[keep], size[keep], spread[keep], keys[keep]), dim, torch.bfloat16)


@pytest.mark.gpu
@pytest.mark.parametrize("lo, hi", [(0, 32), (32, 96), (0, 512), (1408, 1 << 20)], ids=str)
@pytest.mark.parametrize("splits", [1, 2, 5])
@pytest.mark.parametrize("geometry", [(8, 2, 128, 64), (8, 8, 64, 64), (8, 2, 64, 16), (32, 1, 64, 64)], ids=str)
def test_decode(geometry, splits, lo, hi):
    ctx, q, view, dense, bad = spoiled(*geometry, lo, hi)
    heads, kv_heads, dim, _ = geometry
    out = torch.empty(4, heads * dim, dtype=torch.bfloat16, device=DEV)
    ops_tensor.attention(ctx, q, view, out, heads, kv_heads, dim, 0, dim ** -0.5, splits=splits, impl="mma")
    compare(out, ctx, q, dense, bad, heads, kv_heads, dim)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=str)
@pytest.mark.parametrize("sink", [False, True], ids=["", "sink"])
def test_runs_that_are_finished_elsewhere(dtype, sink):
    """Rows of three runs each: all with keys; one of NaN; one without keys; the run of NaN alone with keys."""
    inf, nan = float("inf"), float("nan")
    ml = torch.tensor([[[0.5, 2.0], [1.5, 3.0], [-2.0, 1.0]], [[0.5, 2.0], [-inf, nan], [-2.0, 1.0]],
                       [[0.5, 2.0], [-inf, 0.0], [-2.0, 1.0]], [[-inf, 0.0], [-inf, nan], [-inf, 0.0]]], device=DEV)
    o = torch.randn(4, 3, 16, device=DEV)
    o[1, 1], o[3, 1] = nan, nan
    sinks = torch.tensor([0.25], device=DEV) if sink else None
    out = torch.empty(4, 16, dtype=dtype, device=DEV)
    ops.attention_finish(out, 4, 1, 16, partial=(o, ml, 3), sink_log2=sinks)
    assert torch.isnan(out[1]).all() and torch.isnan(out[3]).all()
    for r in (0, 2):
        w = torch.exp2(ml[r, :, 0].double())
        want = (w[:, None] * o[r].double()).sum(0) / ((w * ml[r, :, 1].double()).sum() + (2.0 ** 0.25 if sink else 0.0))
        assert (out[r].double() - want).abs().max() <= want.abs().max() * (2.0 ** -8 if dtype == torch.bfloat16 else 2.0 ** -19)
