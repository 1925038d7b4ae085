"""Engines whose budget holds everything but the room for shared prefixes: they are built, and their forks read sequence by sequence."""
import numpy as np
import pytest
import torch

from replay_util import TOL_F32
from test_forks import ids, step
from tiny import SHARP, TINY_A, TINY_D, make_model


def engine(d, dtype, **budget):
    from mdma_b200.engine import Engine
    return Engine(d, dtype=dtype, max_batch=6, max_context=256, reserve_mib=0, **budget)


@pytest.mark.gpu
@pytest.mark.parametrize("cfg", [TINY_A, TINY_D], ids="AD")
def test_a_budget_without_room_for_shared_prefixes(cfg):
    from mdma_b200.engine import MemoryBudgetError
    d, _, _ = make_model(cfg, 2, torch.float32, std_scale=SHARP)
    whole = engine(d, "float32")
    most = whole.memory_plan()["total_bytes"]
    small = engine(d, "float32", vram_bytes=most - 1)
    plan = small.memory_plan()
    assert plan["total_bytes"] < most and small.held_bytes()["total_bytes"] == plan["total_bytes"]
    assert plan["kernel_scratch_bytes"] < whole.memory_plan()["kernel_scratch_bytes"]
    with pytest.raises(MemoryBudgetError) as e:
        engine(d, "float32", vram_bytes=plan["total_bytes"] - 1)
    assert e.value.requested == plan["total_bytes"]
    got = []
    for eng in (whole, small):
        a = eng.acquire()
        step(eng, [(a, ids(cfg, 100, 0))])
        slots = [a] + eng.fork(a, 3)
        rows = [step(eng, [(s, ids(cfg, 3, i), [2]) for i, s in enumerate(slots)]),
                step(eng, [(s, [5 + j], [0]) for j, s in enumerate(slots)])]
        session = eng.decode_session()
        session.start(slots, [3] * 4)
        session.run(1)
        rows.append(session.logits[:4].double().cpu().numpy())
        got.append(np.concatenate(rows))
        assert (eng.prefix_groups(slots, [110] * 4, [1] * 4) is None) == (eng is small)
    assert np.abs(got[0] - got[1]).max() <= 2 * TOL_F32 * max(1.0, np.abs(got[0]).max())
    outs = [eng.generate([ids(cfg, 40, 7)], max_tokens=8, n=2)[1].tokens for eng in (whole, small)]
    assert outs[0] == outs[1] and len(outs[0]) == 8


@pytest.mark.gpu
def test_steps_that_gain_nothing_are_steps_without_groups():
    """Forks of a short prompt in bfloat16 are read by every sequence: no tables go up, and the graphs of steps without forks
    serve them."""
    d, _, _ = make_model(TINY_D, 2, torch.bfloat16, std_scale=SHARP)
    eng = engine(d, "bfloat16")
    eng.generate([ids(TINY_D, 40, i) for i in range(4)], max_tokens=6)
    session = eng.decode_session()
    graphs = dict(session.graphs)
    eng.generate([ids(TINY_D, 50, 9)], max_tokens=6, n=4)
    eng.generate([ids(TINY_D, 60, 9)], max_tokens=6, n=2)
    assert all(len(key) == 3 for key in session.graphs) and all(session.graphs[key] is g for key, g in graphs.items())


@pytest.mark.gpu
def test_layers_that_never_share_need_no_groups():
    import gevonex_tiny
    from mdma_b200.engine import Engine
    d = gevonex_tiny.make_model(gevonex_tiny.CFG_A, 3)[0]
    eng = Engine(d, dtype="float32", max_batch=4, max_context=96, page_size=16)
    assert (not eng._sharing) == (not any(getattr(p, "prefix_shapes", list)() for p in eng.model.all_parts()))
    a = eng.acquire()
    step(eng, [(a, list(range(3, 40)), [0])])
    slots = [a] + eng.fork(a, 2)
    assert (eng.prefix_groups(slots, [37] * 3, [1] * 3) is None) == (not eng._sharing)


@pytest.mark.gpu
@pytest.mark.parametrize("page", [16, 64])
def test_small_prefixes_shared_by_force(monkeypatch, page):
    """Whatever pays: prompts and single tokens through the kernels of shared prefixes, on pages of either kind."""
    from mdma_b200 import ops_tensor
    from test_forks import TINY_B, shared_whatever_the_size, test_forked_sequences_against_the_plain_implementation as forked
    plans = shared_whatever_the_size(monkeypatch, 0)
    kinds = set()
    real = ops_tensor.prefix_attention
    monkeypatch.setattr(ops_tensor, "prefix_attention", lambda ctx, *a, **k: (kinds.add(ctx.max_new > 1), real(ctx, *a, **k))[1])
    forked("bfloat16", TINY_B, page)
    assert kinds == {True, False} and plans


@pytest.mark.gpu
@pytest.mark.parametrize("cfg", [TINY_A, TINY_D], ids="AD")
def test_prompts_behind_a_long_prefix(cfg, monkeypatch):
    """Several tokens a sequence behind a prefix that pays by the rule itself, beside a prompt that shares nothing."""
    from mdma_b200 import ops_tensor
    from mdma_b200.engine import Engine
    from plain_llama import plain_forward
    from replay_util import assert_close
    monkeypatch.setattr(ops_tensor, "PREFIX_SHORT", 60)
    d, c, tensors = make_model(cfg, 1, torch.bfloat16, std_scale=SHARP)
    weights = {k: v.float() for k, v in tensors.items()}
    eng = Engine(d, dtype="bfloat16", max_batch=6, max_context=256, logit_rows=8)
    used = []
    real = ops_tensor.prefix_attention
    monkeypatch.setattr(ops_tensor, "prefix_attention", lambda ctx, *a, **k: (used.append(ctx.max_new), real(ctx, *a, **k))[1])
    text = ids(cfg, 70, 0)
    a = eng.acquire()
    step(eng, [(a, text)])
    slots = [a] + eng.fork(a, 2)
    lone = eng.acquire()
    news = [ids(cfg, n, 5 + n) for n in (40, 1, 33, 50)]
    got = step(eng, [(s, t, [len(t) - 1]) for s, t in zip(slots + [lone], news)])
    want = [plain_forward(c, weights, (text if i < 3 else []) + t, torch.float64).numpy()[-1] for i, t in enumerate(news)]
    assert_close(got, np.stack(want), "bfloat16", "prompts")
    assert used == [50] * c.num_hidden_layers if hasattr(c, "num_hidden_layers") else set(used) == {50}
