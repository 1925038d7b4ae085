"""Attention over shared prefixes refuses tables whose layout is not the one that its kernels read."""
from types import SimpleNamespace

import pytest
import torch

from prefix_util import check_close, definition, make_batch
from mdma_b200 import ops, ops_tensor
from mdma_b200.ops import KernelError


def changed(of, **fields):
    return SimpleNamespace(**{**vars(of), **fields})


@pytest.mark.gpu
@pytest.mark.parametrize("fn", [ops.prefix_attention, ops_tensor.prefix_attention], ids=["cuda cores", "tensor cores"])
def test_tables_of_another_layout(fn):
    ctx, q, view, _ = make_batch([(100, [(0, 1), (1, 1), (70, 1)]), (9, [(5, 1)])], 8, 2, 64, 64, torch.bfloat16, 0, "cuda")
    out = torch.full((ctx.n_tokens, 512), 7.0, dtype=q.dtype, device="cuda")
    wide = lambda t: torch.stack([t, t], 1)[:, 0]  # noqa: E731      (every second word of a longer row)
    table = view.page_table
    views = [changed(view, max_pages=view.max_pages + 1), changed(view, max_pages=view.max_pages - 1), changed(view, page_table=table.flatten()),
             changed(view, page_table=table[:, :-1]), changed(view, page_table=table.t().contiguous().t())]
    steps = [changed(ctx, **{f: wide(getattr(ctx, f))}) for f in ("seq_start", "seq_pos0", "seq_slot", "tok_seq")]
    steps += [changed(ctx, prefix=changed(ctx.prefix, **{f: wide(getattr(ctx.prefix, f))})) for f in ("group_len", "tok_first", "toks", "seq_skip")]
    for c, v in [(ctx, v) for v in views] + [(s, view) for s in steps]:
        with pytest.raises(KernelError):
            fn(c, q, v, out, 8, 2, 64, 0.125)
    assert (out == 7.0).all()
    fn(ctx, q, view, out, 8, 2, 64, 0.125)
    assert torch.isfinite(out).all()


@pytest.mark.gpu
@pytest.mark.parametrize("path", ["float32", "bfloat16", "tcgen05", "streamed", "whole lists"])
def test_few_families_among_many_that_share_nothing(path, monkeypatch):
    """The grid has room for the families' tiles, wherever they stand among the groups, and not for a tile a sequence."""
    dtype = torch.float32 if path == "float32" else torch.bfloat16
    new = 3 if path == "whole lists" else 1
    groups = [(0, [(i % 7, new)]) for i in range(40)] + [(100, [(i, new) for i in range(9)])] + [(0, [(70, new)])] + [(65, [(0, new)])] + [(200, [(3, new)] * 30)]
    ctx, q, view, dense = make_batch(groups, 8, 2, 64, 64, dtype, 3, "cuda")
    assert ctx.prefix.n_groups == 44 and ctx.prefix.n_shared == 3
    if path in ("tcgen05", "streamed"):
        monkeypatch.setattr(ops_tensor, "prefix_plan", lambda *a: (2, 1, 0 if path == "tcgen05" else 1))
    order = torch.randperm(44, generator=torch.Generator().manual_seed(1)).tolist()          # families first, last and in between
    host = ctx.prefix._host
    firsts = host["tok_first"].tolist()
    toks = [host["toks"][firsts[g]:firsts[g + 1]] for g in order]
    ints = lambda x: torch.tensor([int(n) for n in x], dtype=torch.int32, device="cuda")  # noqa: E731
    ctx.prefix.group_len, ctx.prefix.group_seq = ints(host["group_len"][g] for g in order), ints(host["group_seq"][g] for g in order)
    ctx.prefix.toks = ints(t for part in toks for t in part)
    ctx.prefix.tok_first = ints([0] + [sum(len(p) for p in toks[:i + 1]) for i in range(44)])
    out = torch.empty(ctx.n_tokens, 512, dtype=dtype, device="cuda")
    (ops if path in ("float32", "bfloat16") else ops_tensor).prefix_attention(ctx, q, view, out, 8, 2, 64, 0.125)
    check_close(out, definition(ctx, q, dense, 8, 2, 64, 0.125), 64, dtype)
