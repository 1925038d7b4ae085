"""Pages whose places lie beyond 2^32 bytes (and 2^31 numbers) of a pool."""
import pytest
import torch

from prefix_util import check_close, definition, make_batch
from mdma_b200 import ops, ops_tensor


@pytest.mark.gpu
@pytest.mark.parametrize("path, plan", [("tensor", (3, 2, 0)), ("tensor", (3, 2, 1)), ("tensor", (3, 2, 2)), ("tensor", (0, 2, 1)), ("whole lists", (2, 0, 0)),
                                        ("float32", (3, 2)), ("bfloat16", (3, 2))], ids=str)
def test_attention_over_far_pages(path, plan, monkeypatch):
    dtype = torch.float32 if path == "float32" else torch.bfloat16
    new = 3 if path == "whole lists" else 1
    heads, kv_heads, dim, ps = 32, 8, 128, 64
    ctx, q, view, dense = make_batch([(300, [(0, new), (70, new), (130, new)]), (0, [(90, new)])], heads, kv_heads, dim, ps, dtype, 6, "cuda")
    n = view.k.shape[0]
    far = 2 ** 31 // (ps * kv_heads * dim) + 1           # numbers beyond 2^31, bytes beyond 2^32
    for name in ("k", "v"):
        pool = torch.empty(far + n, ps, kv_heads, dim, dtype=dtype, device="cuda")
        pool[far:] = getattr(view, name)
        setattr(view, name, pool)
    view.page_table = view.page_table + far
    if path == "tensor" or path == "whole lists":
        monkeypatch.setattr(ops_tensor, "prefix_plan", lambda *a: plan)
    else:
        monkeypatch.setattr(ops, "prefix_plan", lambda *a: plan)
    out = torch.empty(ctx.n_tokens, heads * dim, dtype=dtype, device="cuda")
    (ops if path in ("float32", "bfloat16") else ops_tensor).prefix_attention(ctx, q, view, out, heads, kv_heads, dim, 0.0884)
    check_close(out, definition(ctx, q, dense, heads, kv_heads, dim, 0.0884), dim, dtype)


@pytest.mark.gpu
def test_copies_between_far_pages():
    pages = 2 ** 32 // (64 * 1024) + 9
    pool = torch.zeros(1, pages, 64, 1024, dtype=torch.uint8, device="cuda")
    pool[0, pages - 1], pool[0, 3] = torch.randint(0, 256, (64, 1024), device="cuda", dtype=torch.uint8), 7
    want = pool[0, pages - 1].clone()
    ops.copy_pages([pool], [pages - 1, pages - 1, 3], [pages - 2, 0, pages - 5], [64, 17, 64])
    assert torch.equal(pool[0, pages - 2], want) and torch.equal(pool[0, 0, :17], want[:17]) and not pool[0, 0, 17:].any()
    assert (pool[0, pages - 5] == 7).all() and not pool[0, pages - 4].any() and not pool[0, 1].any()
