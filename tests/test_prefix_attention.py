"""Attention of sequences that share their beginning: the kernels against the definition in 64 bits, and what they refuse."""
from types import SimpleNamespace

import pytest
import torch

from prefix_util import check_close, definition, make_batch, scale_of
from mdma_b200 import ops, ops_tensor
from mdma_b200.cache import PrefixGroups
from mdma_b200.ops import KernelError

DEV = "cuda"


# ---- the groups, on the CPU ---------------------------------------------------------------------------------------------------
def test_groups_cover_every_token_once():
    g = PrefixGroups([(5, [3, 0]), (9, [2])], [7, 3, 9, 5], [1, 4, 2, 3], "cpu")
    assert g.n_groups == 3 and g.group_len.tolist() == [5, 9, 0] and g.group_seq.tolist() == [3, 2, 1]
    assert g.toks.tolist() == [7, 8, 9, 0, 5, 6, 1, 2, 3, 4] and g.tok_first.tolist() == [0, 4, 6, 10]
    assert g.seq_skip.tolist() == [5, 0, 9, 5]
    assert (g.most_tokens, g.most_len, g.most_own) == (4, 9, 7)


@pytest.mark.parametrize("shared, pos0, new", [([(5, [0])], [4], [1]), ([(2, [0, 0])], [4], [1]), ([(2, [0]), (3, [0, 1])], [4, 4], [1, 1]),
                                               ([(2, [1])], [4], [1]), ([(2, [])], [4], [1]), ([(-1, [0])], [4], [1]), ([], [4], [1, 1])])
def test_groups_refuse(shared, pos0, new):
    with pytest.raises(ValueError):
        PrefixGroups(shared, pos0, new, "cpu")


def test_no_cpu_path():
    ctx, q, view, _ = make_batch([(3, [(0, 1)])], 2, 1, 16, 16, torch.float32)
    out = torch.empty(ctx.n_tokens, 32)
    with pytest.raises(KernelError, match="no CPU path"):
        ops.prefix_attention(ctx, q, view, out, 2, 1, 16, 0.25)


# ---- the kernels --------------------------------------------------------------------------------------------------------------
ONE = [(0, 1), (1, 1), (70, 1), (5, 1)]
# (name, groups): prefixes that end inside pages and tiles, prefixes of one token, groups of one, sequences that share nothing
BATCHES = [
    ("one token of one sequence", [(0, [(0, 1)])]),
    ("a prefix of one token", [(1, [(0, 1), (0, 1)])]),
    ("four samples", [(100, ONE)]),
    ("a whole page", [(128, ONE)]),
    ("just over a tile", [(129, [(0, 1)] * 9)]),
    ("groups and loners", [(300, ONE), (0, [(20, 1)]), (7, [(0, 1), (200, 1)]), (0, [(0, 1)]), (64, [(3, 1)])]),
    ("more rows than a tile", [(200, [(i % 5, 1) for i in range(70)])]),
    ("a long prefix, own keys of all lengths", [(1500, [(i * 37 % 400, 1) for i in range(6)])]),
    ("own keys beyond a thousand", [(70, [(1500, 1), (3, 1)]), (0, [(1100, 1)])]),
    ("short prompts", [(131, [(0, 3), (0, 17), (9, 1), (0, 40)])]),
    ("prompts longer than the prefix", [(10, [(0, 150), (3, 77)]), (0, [(0, 130)]), (0, [(5, 2)])]),
    ("prompts and single tokens", [(260, [(0, 1), (0, 65), (129, 1)]), (513, [(0, 9), (1, 64)])]),
]
GEOMETRIES = [(8, 2, 64, 64), (4, 4, 128, 64), (12, 4, 80, 16), (6, 1, 96, 32), (10, 2, 128, 128), (64, 1, 16, 64), (5, 1, 48, 48)]


def run_case(groups, heads, kv_heads, dim, page_size, dtype, simple, sink=False, seed=0, q_gain=1.0, pad=24):
    ctx, q, view, dense = make_batch(groups, heads, kv_heads, dim, page_size, dtype, seed, DEV, pad=pad)
    q = (q.float() * q_gain).to(dtype)
    sinks = torch.linspace(-3, 3, heads, device=DEV) if sink else None
    out = torch.full((ctx.n_tokens + 2, heads * dim), 7.0, dtype=dtype, device=DEV)
    if simple:
        ops.prefix_attention(ctx, q, view, out, heads, kv_heads, dim, scale_of(dim), sinks=sinks)
    else:
        ops_tensor.prefix_attention(ctx, q, view, out, heads, kv_heads, dim, scale_of(dim),
                                    sink_log2=None if sinks is None else sinks * 1.4426950408889634)
        ops_tensor.check_status(q.device)
    assert (out[ctx.n_tokens:] == 7.0).all(), "rows behind the last token were written"
    check_close(out[:ctx.n_tokens], definition(ctx, q, dense, heads, kv_heads, dim, scale_of(dim), sinks), dim, dtype)


@pytest.mark.gpu
@pytest.mark.parametrize("geometry", GEOMETRIES, ids=str)
@pytest.mark.parametrize("name", [n for n, _ in BATCHES])
@pytest.mark.parametrize("path", ["float32", "bfloat16", "tensor"])
def test_against_the_definition(path, name, geometry):
    groups = dict(BATCHES)[name]
    run_case(groups, *geometry, torch.float32 if path == "float32" else torch.bfloat16, path != "tensor", sink=len(name) % 2 == 0)


@pytest.mark.gpu
@pytest.mark.parametrize("geometry", [(3, 1, 33, 64), (2, 2, 256, 16), (8, 2, 20, 64), (80, 1, 128, 64)], ids=str)
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=str)
def test_geometries_of_the_cuda_cores(geometry, dtype):
    run_case(dict(BATCHES)["groups and loners"], *geometry, dtype, True, sink=True)
    run_case(dict(BATCHES)["short prompts"], *geometry, dtype, True)


@pytest.mark.gpu
@pytest.mark.parametrize("path", ["float32", "tensor"])
def test_sharp_scores(path):
    """Queries twelve times as large: the softmax picks a few keys, the running maximum moves often."""
    for name in ("groups and loners", "prompts and single tokens", "a long prefix, own keys of all lengths"):
        run_case(dict(BATCHES)[name], 8, 2, 64, 64, torch.float32 if path == "float32" else torch.bfloat16, path != "tensor", q_gain=12.0)


@pytest.mark.gpu
@pytest.mark.parametrize("path", ["float32", "tensor"])
def test_as_if_nothing_were_shared(path):
    """The same step with the groups and without: within the sum of both bounds (each is checked against the definition)."""
    for share in (True, False):
        ctx, q, view, dense = make_batch([(333, ONE)], 8, 2, 64, 64, torch.float32 if path == "float32" else torch.bfloat16, 3, DEV)
        if not share:
            ctx.prefix = PrefixGroups([], ctx.seq_pos0.tolist(), [1] * 4, DEV)
        out = torch.empty(ctx.n_tokens, 512, dtype=q.dtype, device=DEV)
        (ops if path == "float32" else ops_tensor).prefix_attention(ctx, q, view, out, 8, 2, 64, 0.125)
        check_close(out, definition(ctx, q, dense, 8, 2, 64, 0.125), 64, q.dtype)


@pytest.mark.gpu
@pytest.mark.parametrize("news", [1, 5], ids=["single tokens", "prompts"])
@pytest.mark.parametrize("path", ["float32", "bfloat16", "tensor"])
@pytest.mark.parametrize("geometry", [(8, 2, 64, 64), (4, 4, 128, 16), (4, 1, 32, 32)], ids=str)
def test_what_is_not_finite_stays_with_its_sequence(geometry, path, news):
    """A sequence whose own keys and values hold infinities and NaN gets what its formula gives; the others do not notice."""
    heads, kv_heads, dim, ps = geometry
    dtype = torch.float32 if path == "float32" else torch.bfloat16
    ctx, q, view, dense = make_batch([(130, [(9, news), (0, news), (70, news), (3, news)])], heads, kv_heads, dim, ps, dtype, 5, DEV)
    bad = 2
    pos = int(ctx.seq_pos0[bad])
    page = int(view.page_table[ctx.seq_slot[bad], pos // ps])
    view.k[page, pos % ps] = float("nan")
    view.v[page, pos % ps] = float("inf")
    out = torch.empty(ctx.n_tokens, heads * dim, dtype=dtype, device=DEV)
    (ops_tensor if path == "tensor" else ops).prefix_attention(ctx, q, view, out, heads, kv_heads, dim, scale_of(dim))
    want, size, spread, keys = definition(ctx, q, dense, heads, kv_heads, dim, scale_of(dim))
    keep = torch.tensor([s != bad for s in ctx.tok_seq.tolist()])
    check_close(out.cpu()[keep], (want[keep], size[keep], spread[keep], keys[keep]), dim, dtype)
    a = int(ctx.seq_start[bad])
    assert not torch.isfinite(out[a]).any()


@pytest.mark.gpu
@pytest.mark.parametrize("path", ["float32", "tensor"])
def test_captured_on_another_stream_and_replayed(path):
    """A captured call takes what lies in its tensors at every replay; calls on two streams do not share their parts."""
    dtype = torch.float32 if path == "float32" else torch.bfloat16
    fn = ops.prefix_attention if path == "float32" else ops_tensor.prefix_attention
    cases = [make_batch([(900, [(i, 1) for i in range(20)])], 8, 2, 64, 64, dtype, seed, DEV) for seed in (1, 2)]
    outs = [torch.empty(20, 512, dtype=dtype, device=DEV) for _ in cases]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in cases]
    for _ in range(5):
        for (ctx, q, view, _), out, stream in zip(cases, outs, streams):
            with torch.cuda.stream(stream):
                fn(ctx, q, view, out, 8, 2, 64, 0.125)
    torch.cuda.synchronize()
    for (ctx, q, view, dense), out in zip(cases, outs):
        check_close(out, definition(ctx, q, dense, 8, 2, 64, 0.125), 64, dtype)
    ctx, q, view, dense = cases[0]
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        fn(ctx, q, view, outs[0], 8, 2, 64, 0.125)
    q2 = (torch.randn(q.shape, generator=torch.Generator().manual_seed(9)).to(dtype)).to(DEV)
    q.copy_(q2)
    outs[0].zero_()
    graph.replay()
    check_close(outs[0], definition(ctx, q2, dense, 8, 2, 64, 0.125), 64, dtype)


@pytest.mark.gpu
@pytest.mark.parametrize("plan", [(0, 1, 1), (0, 3, 1), (1, 1, 1), (5, 2, 1), (32, 1, 1), (1, 1, 0), (7, 1, 0), (9, 4, 0), (32, 16, 0), (3, 2, 2), (32, 32, 2)], ids=str)
@pytest.mark.parametrize("geometry", [(8, 2, 64, 64), (32, 2, 128, 64), (3, 1, 96, 128)], ids=str)
def test_every_kernel_and_cut_of_single_tokens(geometry, plan, monkeypatch):
    """Whichever kernel does the prefixes and into however many pieces the keys are cut."""
    monkeypatch.setattr(ops_tensor, "prefix_plan", lambda *a: plan)
    run_case([(1000, ONE), (0, [(300, 1)]), (65, [(0, 1)] * 7)], *geometry, torch.bfloat16, False, sink=True)


@pytest.mark.gpu
@pytest.mark.parametrize("pieces", [1, 2, 5, 32])
def test_every_cut_of_whole_lists(pieces, monkeypatch):
    monkeypatch.setattr(ops_tensor, "prefix_plan", lambda *a: (pieces, 0, 0))
    for name in ("prompts and single tokens", "prompts longer than the prefix", "groups and loners"):
        run_case(dict(BATCHES)[name], 8, 2, 64, 64, torch.bfloat16, False, sink=pieces > 1)
    run_case([(300, [(i % 3, 1 + i % 2) for i in range(200)])], 2, 2, 64, 64, torch.bfloat16, False)       # many sequences a block


@pytest.mark.gpu
@pytest.mark.parametrize("plan", [(1, 1), (32, 32), (3, 2)], ids=str)
def test_every_cut_on_the_cuda_cores(plan, monkeypatch):
    monkeypatch.setattr(ops, "prefix_plan", lambda *a: plan)
    for name in ("groups and loners", "prompts and single tokens"):
        run_case(dict(BATCHES)[name], 6, 2, 72, 16, torch.float32, True, sink=True)


@pytest.mark.gpu
def test_refusals():
    ctx, q, view, _ = make_batch([(100, ONE)], 8, 2, 64, 64, torch.bfloat16, 0, DEV)
    out = torch.empty(ctx.n_tokens, 512, dtype=q.dtype, device=DEV)

    def refused(ctx=ctx, q=q, view=view, out=out, heads=8, kv_heads=2, dim=64, scale=0.125, fn=ops_tensor.prefix_attention, **kw):
        with pytest.raises(KernelError):
            fn(ctx, q, view, out, heads, kv_heads, dim, scale, **kw)
    both = (ops.prefix_attention, ops_tensor.prefix_attention)
    for fn in both:
        refused(fn=fn, heads=7)
        refused(fn=fn, dim=32)
        refused(fn=fn, scale=0.0)
        refused(fn=fn, q=q.float())
        refused(fn=fn, out=out[:, :448])
        refused(fn=fn, out=out[:2])
        refused(fn=fn, out=torch.empty(ctx.n_tokens, 1024, dtype=q.dtype, device=DEV)[:, ::2])
        refused(fn=fn, q=q[:2])
        refused(fn=fn, ctx=SimpleNamespace(**{**vars(ctx), "seq_slot": ctx.seq_slot.long()}))
        refused(fn=fn, ctx=SimpleNamespace(**{**vars(ctx), "n_seqs": ctx.n_seqs + 1}))
        refused(fn=fn, view=SimpleNamespace(**{**vars(view), "k": view.k.transpose(0, 1)}))
        refused(fn=fn, view=SimpleNamespace(**{**vars(view), "page_size": 32}))
    refused(sink_log2=torch.zeros(4, device=DEV))
    refused(fn=ops.prefix_attention, sinks=torch.zeros(8, device=DEV, dtype=torch.bfloat16))
    refused(fn=ops.prefix_attention, scratch=torch.empty(10, device=DEV))
    refused(q=torch.empty(ctx.n_tokens, 516, dtype=q.dtype, device=DEV))           # rows that are not 16-byte aligned
    wide = make_batch([(9, [(0, 1)])], 2, 1, 144, 16, torch.bfloat16, 0, DEV)
    refused(wide[0], wide[1], wide[2], torch.empty(1, 288, dtype=q.dtype, device=DEV), 2, 1, 144, 0.1)
    big = make_batch([(9, [(0, 1)])], 2, 1, 260, 16, torch.bfloat16, 0, DEV)
    refused(big[0], big[1], big[2], torch.empty(1, 520, dtype=q.dtype, device=DEV), 2, 1, 260, 0.1, fn=ops.prefix_attention)
