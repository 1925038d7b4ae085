"""Batches whose sequences share prefixes, for the tests of the kernels: page tables, caches, the definition in 64 bits."""
import math
from types import SimpleNamespace

import torch

from mdma_b200.cache import PrefixGroups

U = {torch.bfloat16: 2.0 ** -8, torch.float32: 2.0 ** -24}     # half a step, relative


def make_batch(groups, heads, kv_heads, dim, page_size, dtype, seed=0, device="cpu", pad=0, poison=float("nan"), order_seed=None):
    """`groups`: (prefix length, [(own tokens held, new tokens), ...]); a prefix of 0 shares nothing.  Every row of the cache that
    belongs to nobody holds `poison`.  `pad`: further columns of a query row."""
    gen = torch.Generator().manual_seed(seed)
    seqs = [(g, length, before, new) for g, (length, members) in enumerate(groups) for before, new in members]
    order = torch.randperm(len(seqs), generator=gen).tolist()
    seqs = [seqs[i] for i in order]
    lengths = [length + before + new for _, length, before, new in seqs]
    ps, max_pages = page_size, max(-(-n // page_size) for n in lengths) + 1
    n_slots = len(seqs) + 3
    n_pages = sum(-(-n // ps) for n in lengths) + sum(length // ps for length, _ in groups) + 3
    free = torch.randperm(n_pages, generator=gen).tolist()
    slots = torch.randperm(n_slots, generator=gen)[:len(seqs)].tolist()
    table = torch.full((n_slots, max_pages), n_pages - 1, dtype=torch.int32)      # (never read: a page that exists)
    k = torch.full((n_pages, ps, kv_heads, dim), poison, dtype=dtype)
    v = torch.full((n_pages, ps, kv_heads, dim), poison, dtype=dtype)
    whole = [[free.pop() for _ in range(length // ps)] for length, _ in groups]
    shared = [(torch.randn(length, kv_heads, dim, generator=gen).to(dtype), torch.randn(length, kv_heads, dim, generator=gen).to(dtype))
              for length, _ in groups]
    dense = []
    for (g, length, before, new), slot, n in zip(seqs, slots, lengths):
        pages = whole[g] + [free.pop() for _ in range(-(-n // ps) - length // ps)]
        table[slot, :len(pages)] = torch.tensor(pages, dtype=torch.int32)
        rows = [torch.cat([part, torch.randn(before + new, kv_heads, dim, generator=gen).to(dtype)]) for part in shared[g]]
        dense.append(rows)
        at = torch.arange(n)
        for pool, row in zip((k, v), rows):
            pool[torch.tensor(pages)[at // ps], at % ps] = row
    news = [new for *_, new in seqs]
    starts = [0]
    for n in news:
        starts.append(starts[-1] + n)
    pos0 = [length + before for _, length, before, _ in seqs]
    q = torch.randn(starts[-1], heads * dim + pad, generator=gen).to(dtype)
    ints = lambda x: torch.tensor(x, dtype=torch.int32, device=device)  # noqa: E731
    shares = [(length, [i for i, s in enumerate(seqs) if s[0] == g]) for g, (length, _) in enumerate(groups) if length]
    ctx = SimpleNamespace(seq_start=ints(starts), seq_pos0=ints(pos0), seq_slot=ints(slots), n_seqs=len(seqs), n_tokens=starts[-1],
                          tok_seq=ints([i for i, n in enumerate(news) for _ in range(n)]),
                          tok_pos=ints([p + t for p, n in zip(pos0, news) for t in range(n)]),
                          max_new=max(news), max_len=max(lengths), prefix=PrefixGroups(shares, pos0, news, device))
    view = SimpleNamespace(k=k.to(device), v=v.to(device), page_table=table.to(device), page_size=ps, max_pages=max_pages)
    return ctx, q.to(device), view, dense


def definition(ctx, q, dense, heads, kv_heads, dim, scale, sinks=None):
    """(result, sum of |weight * value|, largest sum over |q_d k_d| * scale, most keys) per token and head, in 64 bits."""
    q = q.cpu()[:, :heads * dim].double().reshape(-1, heads, dim)
    out = torch.empty(ctx.n_tokens, heads, dim, dtype=torch.float64)
    size = torch.empty_like(out)
    spread = torch.zeros(ctx.n_tokens, heads, 1, dtype=torch.float64)
    keys = torch.zeros(ctx.n_tokens, 1, 1, dtype=torch.float64)
    group = heads // kv_heads
    starts, pos0 = ctx.seq_start.tolist(), ctx.seq_pos0.tolist()
    for i in range(ctx.n_seqs):
        a, b = starts[i], starts[i + 1]
        n = pos0[i] + b - a
        k, v = (x[:n].double().repeat_interleave(group, 1) for x in dense[i])
        s = torch.einsum("thd,nhd->thn", q[a:b], k) * scale
        visible = torch.arange(n)[None, :] <= (pos0[i] + torch.arange(b - a))[:, None]
        s = s.masked_fill(~visible[:, None, :], -math.inf)
        top = s.amax(2, keepdim=True)
        if sinks is not None:
            top = torch.maximum(top, sinks.double().cpu()[None, :, None])
        e = torch.exp(s - top)
        w = e / (e.sum(2, keepdim=True) + (0 if sinks is None else torch.exp(sinks.double().cpu()[None, :, None] - top)))
        out[a:b] = torch.einsum("thn,nhd->thd", w, v)
        size[a:b] = torch.einsum("thn,nhd->thd", w, v.abs())
        spread[a:b] = torch.einsum("thd,nhd->thn", q[a:b].abs(), k.abs()).amax(2, keepdim=True) * scale
        keys[a:b, 0, 0] = pos0[i] + 1.0 + torch.arange(b - a)
    return out, size, spread, keys


def bound_of(want, size, spread, keys, dim, dtype):
    """How far a result may be, number for number.  A score is a sum of dim products and three more roundings in float, each at
    most 2^-24 of sum |q k| * scale: its weight changes by the factor e^d with d below (dim + 8) 2^-24 of that (twice: a
    row's sum has it too); an exponential is off by 2 steps, the sums over the keys and their joining by 2^-24 a
    term.  In bfloat16 every weight is rounded for the second product and the result once more, 2^-8 each."""
    d = (dim + 8) * 2.0 ** -24 * spread
    rel = 2 * torch.expm1(d) + (keys + 64) * 2.0 ** -23
    if dtype == torch.bfloat16:
        rel = rel + U[dtype]
    return size * rel + want.abs() * U[dtype] * 1.01 + 1e-37


def check_close(got, ref, dim, dtype, what=""):
    want, size, spread, keys = ref
    got = got.double().cpu().reshape(want.shape)
    assert torch.isfinite(got).all(), f"{what}: a value is not finite"
    over = (got - want).abs() / bound_of(want, size, spread, keys, dim, dtype)
    assert over.max() <= 1.0, f"{what}: {over.max().item():.2f} times the bound, error {(got - want).abs().max().item():.3g}"


def scale_of(dim):
    return 1.0 / math.sqrt(dim)
