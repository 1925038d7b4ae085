"""A sequence's logits stay as they are, bit for bit, when members of its family end."""
import numpy as np
import pytest
import torch

from prefix_util import check_close, definition, make_batch
from test_forks import ids, shared_whatever_the_size, step
from tiny import SHARP, TINY_D, make_model
from mdma_b200 import ops_tensor


def logits_of(dtype, live, before, own, monkeypatch, slots=6, replayed=False):
    """The first two sequences' logits of single-token steps: a prompt of `before` tokens forks, member i brings own[i] tokens, then
    live[t] sequences are left of it in step t."""
    from mdma_b200.engine import Engine
    d, _, _ = make_model(TINY_D, 2, torch.bfloat16, std_scale=SHARP)
    eng = Engine(d, dtype=dtype, max_batch=slots, max_context=2304)
    a = eng.acquire()
    step(eng, [(a, ids(TINY_D, before, 0))])
    members = [a] + eng.fork(a, len(own) - 1)
    for i, (s, n) in enumerate(zip(members, own)):
        if n:
            step(eng, [(s, ids(TINY_D, n, 10 + i))])
    out = []
    for turn, n in enumerate(live):
        for s in members[n:]:
            eng.release(s)
        members = members[:n]
        if replayed:
            session = eng.decode_session()
            session.start(members, [9 + turn] * n)
            session.run(1)
            session.read()
            out.append(session.logits[:2].double().cpu().numpy())
        else:
            out.append(step(eng, [(s, [9 + turn], [0]) for s in members])[:2])
    return out


@pytest.mark.gpu
@pytest.mark.parametrize("replayed", [False, True], ids=["", "replayed"])
def test_rows_of_a_tile_on_the_cuda_cores(replayed, monkeypatch):
    """Six members of two query heads a kv head, then four, then two: a tile of 32 rows would do at first, one of 8 later."""
    runs = [logits_of("float32", live, 1021, [0] * 6, monkeypatch, replayed=replayed) for live in ([6, 6, 6], [6, 4, 2], [2, 2, 2])]
    for other in runs[1:]:
        assert all(np.array_equal(x, y) for x, y in zip(runs[0], other))


@pytest.mark.gpu
@pytest.mark.parametrize("path", ["float32", "tcgen05", "streamed"])
def test_the_longest_member_ends(path, monkeypatch):
    """The longest of the own keys, beyond a thousand, ends: the others' own keys are cut where they were."""
    if path != "float32":
        shared_whatever_the_size(monkeypatch, 0 if path == "tcgen05" else 1 << 20)
    own = [700, 300, 0, 5, 2100]
    runs = [logits_of("float32" if path == "float32" else "bfloat16", live, 130, own, monkeypatch) for live in ([5, 5, 5], [5, 4, 4], [4, 4, 2])]
    for other in runs[1:]:
        assert all(np.array_equal(x, y) for x, y in zip(runs[0], other))


# ---- how own keys are cut ---------------------------------------------------------------------------------------------------------
def meta(live, most_seqs, most_len):
    from types import SimpleNamespace
    return SimpleNamespace(max_new=1, n_seqs=live, n_tokens=live, most_seqs=most_seqs, most_len=most_len)


@pytest.mark.parametrize("most_len", [500, 4096, 32768, 131072])
@pytest.mark.parametrize("most_seqs", [1, 8, 24, 64, 300, 2000])
def test_the_length_of_a_piece_follows_from_the_engine(most_seqs, most_len):
    """One length, whoever lives; pieces cover every sequence; a long sequence is cut even in a large engine."""
    lengths = set()
    for live in (1, 2, most_seqs):
        for own in (1, 20, 1024, 1025, most_len // 2 + 1, most_len):
            pieces, keys = ops_tensor.prefix_own_cut(meta(live, most_seqs, most_len), min(own, most_len), 8, 148)
            lengths.add(keys)
            assert 1 <= pieces <= 16 and pieces * keys >= min(own, most_len) and (pieces - 1) * keys < own
            assert pieces * most_seqs <= max(most_seqs, ops_tensor.PREFIX_OWN_PARTS)
    assert len(lengths) == 1 and lengths.pop() % 1024 == 0
    if most_seqs <= 64 and most_len == 32768:
        assert ops_tensor.prefix_own_cut(meta(5, most_seqs, most_len), 30000, 8, 148)[0] >= 7


@pytest.mark.parametrize("heads, kv_heads, page", [(32, 8, 64), (32, 32, 64), (64, 2, 64), (8, 2, 16), (8, 8, 32)])
def test_plans_do_not_follow_from_the_longest_sequence(heads, kv_heads, page):
    """Whatever the longest of the live own keys: the prefix's pieces and kernel, and the own keys' pieces where they are not of a fixed
    length."""
    from types import SimpleNamespace
    plans = set()
    for own in (20, 900, 1500, 9000):
        g = SimpleNamespace(most_len=8192, most_own=own, most_tokens=12, n_groups=1, n_shared=1, most_members=12)
        pieces, cut, kind = ops_tensor.prefix_plan(meta(12, 12, 20000), g, heads, kv_heads, 128, 148, page)
        plans.add((pieces, kind, None if ops_tensor.prefix_streams(meta(12, 12, 20000), heads // kv_heads, page) else cut))
    assert len(plans) == 1


@pytest.mark.gpu
@pytest.mark.parametrize("kind", [0, 1], ids=["tcgen05", "streamed"])
def test_pieces_of_a_fixed_length(kind, monkeypatch):
    """Against the definition in pieces of 128 keys; bit for bit the same whether a step has room for the pieces of its longest sequence,
    or for many more; and right if it has been given too few."""
    monkeypatch.setattr(ops_tensor, "PREFIX_OWN_KEYS", 512)
    ctx, q, view, dense = make_batch([(200, [(0, 1), (127, 1), (128, 1), (1, 1)]), (0, [(500, 1), (5, 1)])], 8, 2, 64, 64, torch.bfloat16, 4, "cuda")
    ref = definition(ctx, q, dense, 8, 2, 64, 0.125)
    ctx.most_seqs = 16                                # (their 32 blocks: pieces of a quarter)
    outs, longest = [], ctx.prefix.most_own
    for most_own in (longest, longest + 300, 40):
        ctx.prefix.most_own = most_own
        own, keys = ops_tensor.prefix_own_cut(ctx, most_own, 2, 148)
        assert keys == 128 and own == {longest: 4, longest + 300: 7, 40: 1}[most_own]
        monkeypatch.setattr(ops_tensor, "prefix_plan", lambda *a: (3, own, kind))
        out = torch.empty(ctx.n_tokens, 512, dtype=torch.bfloat16, device="cuda")
        ops_tensor.prefix_attention(ctx, q, view, out, 8, 2, 64, 0.125)
        ops_tensor.check_status(q.device)
        check_close(out, ref, 64, torch.bfloat16, f"{own} pieces")
        outs.append(out)
    assert torch.equal(outs[0], outs[1])
    short = [i for i in range(ctx.n_seqs) if int(ctx.seq_pos0[i]) + 1 - int(ctx.prefix.seq_skip[i]) <= 128]
    assert len(short) == 4 and torch.equal(outs[0][short], outs[2][short])


@pytest.mark.gpu
@pytest.mark.parametrize("path", ["float32", "tcgen05", "streamed"])
def test_runs_across_a_piece_of_own_keys(path, monkeypatch):
    """Replayed runs in which the longest own keys pass 1,024 and a piece's end, bit for bit the steps on their own."""
    from mdma_b200.engine import Engine
    if path != "float32":
        shared_whatever_the_size(monkeypatch, 0 if path == "tcgen05" else 1 << 20)
        monkeypatch.setattr(ops_tensor, "PREFIX_OWN_KEYS", 2048)
    d, _, _ = make_model(TINY_D, 2, torch.bfloat16, std_scale=SHARP)
    out = []
    for replayed in (True, False):
        eng = Engine(d, dtype="float32" if path == "float32" else "bfloat16", max_batch=6, max_context=2304)
        a = eng.acquire()
        step(eng, [(a, ids(TINY_D, 70, 0))])
        slots = [a] + eng.fork(a, 2)
        step(eng, [(a, ids(TINY_D, 1020, 1)), (slots[1], ids(TINY_D, 40, 2))])
        tokens, logits, chosen = [3, 4, 5], {}, []
        if replayed:
            session = eng.decode_session()
            session.start(slots, tokens)
            while len(chosen) < 12:
                session.run(5)
                chosen += [t for t, _ in session.read()]
                logits[len(chosen)] = session.logits[:3].clone()
        else:
            for i in range(12):
                rows = eng.step([(s, [t], [0]) for s, t in zip(slots, tokens)])
                logits[i + 1] = rows.clone()
                tokens = eng.sampler.sample(rows, eng.decode_session().params, [0, 1, 2], [0] * 3)[0]
                chosen.append(tokens)
        eng.check_status()
        out.append((logits, chosen[:12]))
    (replays, picked), (steps, alone) = out
    assert picked == alone and any(n <= 4 for n in replays)          # (a run ended where the own keys reached 1,024)
    assert all(torch.equal(rows, steps[n]) for n, rows in replays.items() if n in steps)
