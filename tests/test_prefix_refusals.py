"""Attention over shared prefixes refuses tables whose layout is not the one that its kernels read."""
from types import SimpleNamespace

import pytest
import torch

from prefix_util import make_batch
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
