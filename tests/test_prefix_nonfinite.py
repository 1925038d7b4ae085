"""Attention over shared prefixes where keys or queries are not finite: NaN comes out where the definition has NaN, and nowhere else."""
import pytest
import torch

from prefix_util import check_close, definition, make_batch, scale_of
from mdma_b200 import ops, ops_tensor
from mdma_b200.cache import PrefixGroups

DEV = "cuda"
NAN = float("nan")
SINGLE = [(1000, [(0, 1), (1, 1), (70, 1), (300, 1)]), (0, [(300, 1)]), (65, [(0, 1)] * 3)]
PROMPTS = [(1000, [(0, 3), (9, 40)]), (0, [(300, 5)]), (65, [(0, 1), (2, 70)])]
# (pieces of a prefix, pieces of own keys, kernel of the prefixes)
TENSOR_SINGLE = [(0, 1, 1), (0, 3, 1), (1, 1, 1), (5, 2, 1), (1, 1, 0), (7, 1, 0), (9, 4, 0), (3, 2, 2)]
TENSOR_PROMPTS = [(1, 0, 0), (5, 0, 0), (3, 2, 2)]


def spoil_keys(view, ctx, dense, seqs, lo, hi):
    """Keys [lo, hi) of these sequences become NaN, in their pages and in the dense rows of the definition."""
    ps = view.page_size
    for i in seqs:
        at = torch.arange(lo, min(hi, dense[i][0].shape[0]))
        pages = view.page_table[int(ctx.seq_slot[i])].cpu().long()[at // ps]
        view.k[pages.to(DEV), (at % ps).to(DEV)] = NAN
        dense[i][0][at] = NAN


def compare(path, groups, geometry, spoil, sink, dtype):
    heads, kv_heads, dim, ps = geometry
    ctx, q, view, dense = make_batch(groups, heads, kv_heads, dim, ps, dtype, 11, DEV, pad=8)
    skip = ctx.prefix.seq_skip.tolist()
    first = [i for i, n in enumerate(skip) if n == groups[0][0]]         # the members of the first group
    if spoil == "prefix":
        spoil_keys(view, ctx, dense, first, 0, groups[0][0])
    elif spoil == "its beginning":
        spoil_keys(view, ctx, dense, first, 0, 512)
    elif spoil == "its end":
        spoil_keys(view, ctx, dense, first, 768, groups[0][0])
    elif spoil == "own keys":
        spoil_keys(view, ctx, dense, first[1:2], groups[0][0], 1 << 30)
    else:
        q[int(ctx.seq_start[first[0]])] = NAN
    sinks = torch.linspace(-3, 3, heads, device=DEV) if sink else None
    out = torch.full((ctx.n_tokens, heads * dim), 7.0, dtype=dtype, device=DEV)
    if path == "tensor":
        ops_tensor.prefix_attention(ctx, q, view, out, heads, kv_heads, dim, scale_of(dim),
                                    sink_log2=None if sinks is None else sinks * 1.4426950408889634)
        ops_tensor.check_status(q.device)
    else:
        ops.prefix_attention(ctx, q, view, out, heads, kv_heads, dim, scale_of(dim), sinks=sinks)
    want, size, spread, keys = definition(ctx, q, dense, heads, kv_heads, dim, scale_of(dim), sinks)
    got = out.double().cpu().reshape(want.shape)
    assert torch.isnan(want).any() and not torch.isnan(want).all()
    assert torch.equal(torch.isnan(got), torch.isnan(want)), f"{int(torch.isnan(got).sum())} NaN, {int(torch.isnan(want).sum())} by the definition"
    keep = ~torch.isnan(want).any(2).any(1)
    check_close(got[keep], (want[keep], size[keep], spread[keep], keys[keep]), dim, dtype)


SPOILS = ["prefix", "its beginning", "its end", "own keys", "a query"]


@pytest.mark.gpu
@pytest.mark.parametrize("sink", [False, True], ids=["", "sink"])
@pytest.mark.parametrize("spoil", SPOILS)
@pytest.mark.parametrize("plan", TENSOR_SINGLE, ids=str)
def test_single_tokens_on_the_tensor_cores(plan, spoil, sink, monkeypatch):
    monkeypatch.setattr(ops_tensor, "prefix_plan", lambda *a: plan)
    compare("tensor", SINGLE, (8, 2, 64, 64), spoil, sink, torch.bfloat16)


@pytest.mark.gpu
@pytest.mark.parametrize("sink", [False, True], ids=["", "sink"])
@pytest.mark.parametrize("spoil", SPOILS)
@pytest.mark.parametrize("plan", TENSOR_PROMPTS, ids=str)
def test_prompts_on_the_tensor_cores(plan, spoil, sink, monkeypatch):
    monkeypatch.setattr(ops_tensor, "prefix_plan", lambda *a: plan)
    compare("tensor", PROMPTS, (4, 1, 128, 64), spoil, sink, torch.bfloat16)


@pytest.mark.gpu
@pytest.mark.parametrize("spoil", SPOILS)
@pytest.mark.parametrize("plan", [(1, 1), (5, 2), (32, 32)], ids=str)
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=str)
def test_on_the_cuda_cores(dtype, plan, spoil, monkeypatch):
    monkeypatch.setattr(ops, "prefix_plan", lambda *a: plan)
    for groups in (SINGLE, PROMPTS):
        compare("simple", groups, (6, 2, 72, 16), spoil, plan[0] > 1, dtype)


@pytest.mark.gpu
@pytest.mark.parametrize("path", ["float32", "tensor"])
def test_a_step_that_shares_nothing(path):
    """Groups of one: what a sequence's own keys alone give."""
    dtype = torch.float32 if path == "float32" else torch.bfloat16
    ctx, q, view, dense = make_batch([(0, [(100, 1), (0, 1)])], 4, 2, 64, 64, dtype, 2, DEV)
    ctx.prefix = PrefixGroups([], ctx.seq_pos0.tolist(), [1, 1], DEV)
    spoil_keys(view, ctx, dense, [0], 0, 1 << 30)
    out = torch.empty(2, 256, dtype=dtype, device=DEV)
    (ops if path == "float32" else ops_tensor).prefix_attention(ctx, q, view, out, 4, 2, 64, 0.125)
    assert torch.isnan(out[0]).all() and torch.isfinite(out[1]).all()
