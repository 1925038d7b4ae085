"""Sequences that fork: engine steps, replayed decode, generation and the command line, with what they share kept and read once."""
import json
import os
import subprocess
import sys

import numpy as np
import pytest
import torch

import degavik_tiny
import fizadra_tiny
import gevonex_tiny
import mogevik_tiny
import salipel_tiny
import tubusun_tiny
from plain_llama import plain_forward, plain_generate
from replay_util import TOL_F32, assert_close
from tiny import SHARP, TINY_A, TINY_B, TINY_C, TINY_D, TINY_E, make_model

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def ids(cfg, n, seed):
    g = torch.Generator().manual_seed(seed)
    return torch.randint(0, cfg["vocab_size"], (n,), generator=g).tolist()


# ---- the loop, on the CPU -----------------------------------------------------------------------------------------------------
class FakeEngine:
    """Counts what it is asked; logits are numbers of sequences."""

    def __init__(self, slots, pages, page_size=4, max_context=64):
        self.max_slots, self.n_pages, self.page_size, self.max_context = slots, pages, page_size, max_context
        self.free, self.live, self.most, self.prompts, self.forks = list(range(slots)), {}, 0, [], []

    def fits(self, sizes):
        from mdma_b200.engine.step import Engine
        self.cache = self                                    # (the pages' count is looked up there)
        return Engine.fits(self, sizes)

    def acquire(self):
        slot = self.free.pop(0)
        self.live[slot] = 0
        self.most = max(self.most, len(self.live))
        return slot

    def release(self, slot):
        del self.live[slot]
        self.free.append(slot)

    def fork(self, slot, n):
        self.forks.append((slot, n))
        new = [self.acquire() for _ in range(n)]
        for s in new:
            self.live[s] = self.live[slot]
        return new

    def fan_out(self, logits, counts):
        return [row for row, n in zip(logits, counts) for _ in range(n)]

    def step(self, entries):
        for e in entries:
            if self.live[e.slot] == 0:
                self.prompts.append(list(e.tokens))
            self.live[e.slot] += len(e.tokens)
        return [sum(e.tokens) for e in entries]


class FakeSampler:
    def sample(self, logits, params, requests, steps, histories=None):
        return [(row * 7 + r * 3 + s) % 50 for row, r, s in zip(logits, requests, steps)], [0] * len(logits)


def test_every_prompt_is_computed_once_and_its_completions_go_on_alone():
    from mdma_b200.engine.generate import Generator
    engine = FakeEngine(8, 100)
    outs = Generator(engine, FakeSampler(), use_graphs=False).generate([[1, 2, 3], [4]], 5, n=4)
    assert engine.prompts == [[1, 2, 3], [4]] and [n for _, n in engine.forks] == [3, 3] and not engine.live
    alone = FakeEngine(8, 100)
    want = Generator(alone, FakeSampler(), use_graphs=False).generate([[1, 2, 3]] * 4 + [[4]] * 4, 5)
    assert [(o.prompt_tokens, o.tokens, o.finish_reason) for o in outs] == [(o.prompt_tokens, o.tokens, o.finish_reason) for o in want]


@pytest.mark.parametrize("slots, pages, most", [(3, 100, 3), (8, 6, 4), (1, 100, 1)])
def test_more_completions_than_fit_take_turns(slots, pages, most):
    from mdma_b200.engine.generate import Generator
    engine = FakeEngine(slots, pages)
    outs = Generator(engine, FakeSampler(), use_graphs=False).generate([list(range(1, 10))], 4, n=7)      # 9 + 3 rows: two shared pages and one each
    assert len(outs) == 7 and engine.most <= most and not engine.live
    assert [o.tokens for o in outs] == [o.tokens for o in Generator(FakeEngine(7, 100), FakeSampler(), use_graphs=False).generate([list(range(1, 10))] * 7, 4)]


def test_no_completion_is_refused():
    from mdma_b200.engine.generate import Generator
    with pytest.raises(ValueError):
        Generator(FakeEngine(2, 9), FakeSampler()).generate([[1]], 2, n=0)


# ---- plans, on the CPU --------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("heads, kv_heads, dim", [(32, 8, 128), (32, 32, 128), (64, 8, 64), (16, 1, 64), (100, 100, 128), (40, 2, 80)])
@pytest.mark.parametrize("page", [16, 32, 64, 128])
@pytest.mark.parametrize("slots", [1, 4, 24, 64, 300])
def test_planned_scratch_takes_every_plan(heads, kv_heads, dim, page, slots):
    """Whatever lengths and families a step of single tokens has, its parts fit what the engine planned; and they do not follow
    from who is left of a family."""
    from types import SimpleNamespace

    from mdma_b200 import ops, ops_tensor
    from mdma_b200.engine.step import prefix_floats
    context = 20000
    part = SimpleNamespace(prefix_shapes=lambda: [(heads, kv_heads, dim)])
    have = prefix_floats(SimpleNamespace(all_parts=lambda: [part]), torch.bfloat16, 148, slots, context, page)
    for length in (1024, 2048, 4096, 10240, context):
        for families in (1, 2, 3, 7, 16, 100):
            for members in (1, 2, 5, 16, 100):
                if families * members > slots:
                    continue
                g = SimpleNamespace(most_len=length, most_own=context, most_tokens=members, n_groups=families, n_shared=families,
                                    most_members=members)
                live = slots - slots // 2
                ctx = SimpleNamespace(max_new=1, n_seqs=slots, n_tokens=slots, most_seqs=slots)
                fewer = SimpleNamespace(max_new=1, n_seqs=live, n_tokens=live, most_seqs=slots)
                plan = ops_tensor.prefix_plan(ctx, g, heads, kv_heads, dim, 148, page)
                assert 0 <= plan[0] <= 32 and 0 <= plan[1] <= 32
                assert ops.prefix_scratch_floats(slots, heads, plan[0] + plan[1], dim) <= have
                g.most_tokens = 1
                assert ops_tensor.prefix_plan(fewer, g, heads, kv_heads, dim, 148, page) == plan


# ---- the engine -----------------------------------------------------------------------------------------------------------------
def step(eng, entries):
    from mdma_b200.engine import StepEntry
    out = eng.step([StepEntry(*e) for e in entries]).double().cpu().numpy()
    eng.check_status()
    return out


@pytest.mark.gpu
@pytest.mark.parametrize("page", [16, 64])
@pytest.mark.parametrize("cfg", [TINY_A, TINY_B, TINY_C, TINY_D, TINY_E], ids="ABCDE")
@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
def test_forked_sequences_against_the_plain_implementation(dtype, cfg, page):
    """A prompt forks into five, which bring a token each, then several, then a token each again; one forks once more, others
    end; every row nobody owns holds NaN."""
    from mdma_b200.engine import Engine
    d, c, tensors = make_model(cfg, 1, torch.bfloat16, std_scale=SHARP)
    weights = {k: v.float() for k, v in tensors.items()}
    eng = Engine(d, dtype=dtype, max_batch=8, max_context=128, page_size=page, logit_rows=64)
    text = {}
    a = eng.acquire()
    text[a] = ids(cfg, 75, 0)
    loner = eng.acquire()
    text[loner] = ids(cfg, 9, 1)
    step(eng, [(a, text[a]), (loner, text[loner])])
    for s in eng.fork(a, 4):
        text[s] = list(text[a])
    pages = eng.cache.n_pages - eng.cache.groups[0].pages.free_count
    assert pages == 75 // page + 5 * (75 % page > 0) + -(-9 // page)
    for turn, news in enumerate([[1] * 8, [3, 1, 7, 2, 5, 1, 1, 1], [1] * 8, [1] * 8]):
        eng.cache.poison_unused()
        if turn == 2:
            (s,) = eng.fork(a)
            text[s] = list(text[a])
            gone = [s for s in text if s not in (a, loner)][0]
            eng.release(gone)
            del text[gone]
        entries, want = [], []
        for s, n in zip(list(text), news):
            tok = ids(cfg, n, 100 * turn + s)
            entries.append((s, tok, list(range(n))))
            text[s] = text[s] + tok
            ref = plain_forward(c, weights, text[s], torch.float64).numpy()
            want.append(ref[-n:])
        got = step(eng, entries)
        assert_close(got, np.concatenate(want), dtype, f"turn {turn}")
        eng.cache.check()
    assert eng.cache.compact() >= 0
    got = step(eng, [(s, [5], [0]) for s in text])
    assert_close(got, np.stack([plain_forward(c, weights, text[s] + [5], torch.float64).numpy()[-1] for s in text]), dtype, "compacted")


OTHERS = [("gevonex", gevonex_tiny, "CFG_A"), ("gevonex", gevonex_tiny, "CFG_B"), ("mogevik", mogevik_tiny, "CFG_A"), ("mogevik", mogevik_tiny, "CFG_B"),
          ("tubusun", tubusun_tiny, "CFG_A"), ("tubusun", tubusun_tiny, "CFG_B"), ("fizadra", fizadra_tiny, "CFG_A"),
          ("fizadra", fizadra_tiny, "CFG_B"), ("degavik", degavik_tiny, "CFG_A"), ("salipel", salipel_tiny, "CFG_A"), ("salipel", salipel_tiny, "CFG_C")]


@pytest.mark.gpu
@pytest.mark.parametrize("name, module, which", OTHERS, ids=[f"{n}-{w}" for n, _, w in OTHERS])
def test_other_architectures_fork(name, module, which):
    """State, windows, chunks, latents: a fork goes on as a sequence that brought the same tokens itself.  Both are within the oracle
    tests' tolerance of the oracle, so within twice that of one another."""
    from mdma_b200.engine import Engine
    made = getattr(module, which)
    d = module.make_model(made, degavik_tiny.RANKS_A, 3)[0] if module is degavik_tiny else module.make_model(made, 3)[0]
    eng = Engine(d, dtype="float32", max_batch=4, max_context=96, page_size=16, logit_rows=64)
    text = torch.randint(0, eng.vocab_size, (60,), generator=torch.Generator().manual_seed(2)).tolist()
    a = eng.acquire()
    step(eng, [(a, text[:37])])
    b, gone = eng.fork(a, 2)
    eng.release(gone)
    eng.cache.poison_unused()
    step(eng, [(a, text[40:44])])
    got = [step(eng, [(b, text[37:45], list(range(8)))]), step(eng, [(b, text[45:46], [0]), (a, text[0:1])])]
    eng.cache.check()
    c = eng.acquire()
    step(eng, [(c, text[:37])])
    want = [step(eng, [(c, text[37:45], list(range(8)))]), step(eng, [(c, text[45:46], [0])])]
    for x, y in zip(got, want):
        assert np.abs(x - y).max() <= 2 * TOL_F32 * max(1.0, np.abs(y).max())


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
def test_replayed_steps_equal_steps_on_their_own(dtype):
    from mdma_b200.engine import Engine
    d, c, _ = make_model(TINY_D, 2, torch.bfloat16, std_scale=SHARP)
    runs = (1, 5, 1, 2)                                # steps a run; the longer sequences pass 1,024 tokens in the second
    steps = {}
    for graphs in (True, False):
        eng = Engine(d, dtype=dtype, max_batch=6, max_context=2304)
        a, b = eng.acquire(), eng.acquire()
        step(eng, [(a, ids(TINY_D, 1021, 0)), (b, ids(TINY_D, 300, 1))])
        slots, tokens = [a, b] + eng.fork(a, 3) + eng.fork(b, 1), [3, 4, 5, 6, 7, 8]
        session = eng.decode_session()
        logits, chosen = {}, []
        if graphs:
            session.start(slots, tokens)
            for n in runs:
                done = session.run(n)
                chosen += [t for t, _ in session.read()]
                assert len(chosen) >= done >= 1
                logits[len(chosen)] = session.logits[:6].clone()
        else:
            for i in range(sum(runs)):
                out = eng.step([(s, [t], [0]) for s, t in zip(slots, tokens)])
                logits[i + 1] = out.clone()
                tokens = eng.sampler.sample(out, session.params, list(range(6)), [0] * 6)[0]
                chosen.append(tokens)
        steps[graphs] = logits, chosen
        eng.check_status()
    replayed, chosen = steps[True]
    assert chosen == steps[False][1][:len(chosen)] and len(replayed) == len(runs)
    for n, logits in replayed.items():
        assert torch.equal(logits, steps[False][0][n])


def shared_whatever_the_size(monkeypatch, rows):
    """Prefixes of any size are shared in bfloat16, those of up to `rows` query rows streamed; returns the plans that are made."""
    from mdma_b200 import ops_tensor
    plans, plan_of = [], ops_tensor.prefix_plan
    monkeypatch.setattr(ops_tensor, "PREFIX_LEAST_BYTES", 0)
    monkeypatch.setattr(ops_tensor, "PREFIX_STREAM_ROWS", rows)

    def noted(ctx, *args):
        plans.append((ctx.max_new, plan_of(ctx, *args)))
        return plans[-1][1]
    monkeypatch.setattr(ops_tensor, "prefix_plan", noted)
    return plans


@pytest.mark.gpu
@pytest.mark.parametrize("rows", [0, 1 << 20], ids=["tcgen05", "streamed"])
@pytest.mark.parametrize("cfg", [TINY_A, TINY_B, TINY_C, TINY_D, TINY_E], ids="ABCDE")
def test_small_prefixes_through_the_kernels_of_large_ones(monkeypatch, cfg, rows):
    plans = shared_whatever_the_size(monkeypatch, rows)
    test_forked_sequences_against_the_plain_implementation("bfloat16", cfg, 64)
    from mdma_b200 import ops_tensor
    if ops_tensor.attention_supported(cfg["num_attention_heads"], cfg["num_key_value_heads"], cfg["head_dim"]):
        group = cfg["num_attention_heads"] // cfg["num_key_value_heads"]
        want = ops_tensor.PREFIX_STREAM if rows and group <= 16 else ops_tensor.PREFIX_TC
        assert any(new == 1 and plan[0] > 0 and plan[2] == want for new, plan in plans)


@pytest.mark.gpu
@pytest.mark.parametrize("rows", [0, 1 << 20], ids=["tcgen05", "streamed"])
def test_replayed_steps_through_the_kernels_of_large_prefixes(monkeypatch, rows):
    plans = shared_whatever_the_size(monkeypatch, rows)
    test_replayed_steps_equal_steps_on_their_own("bfloat16")
    assert any(plan[0] > 0 for _, plan in plans)


@pytest.mark.gpu
def test_graphs_of_families_are_kept_within_bounds():
    """Families of every size in turn, twice: the tokens are those of steps without graphs."""
    from mdma_b200.engine import Engine
    d, c, _ = make_model(TINY_D, 2, torch.bfloat16, std_scale=SHARP)
    eng = Engine(d, dtype="float32", max_batch=6, max_context=256)
    session = eng.decode_session()
    session.most_prefix_graphs = 2
    tokens = {}
    for use_graph in (True, True, False):
        for n in (1, 2, 3, 4, 5):
            a = eng.acquire()
            step(eng, [(a, ids(TINY_D, 70, n))])
            slots = [a] + eng.fork(a, n)
            session.start(slots, [3] * (n + 1))
            got = []
            while len(got) < 4:
                session.run(1, use_graph=use_graph)
                got += [t for t, _ in session.read()]
            for s in slots:
                eng.release(s)
            assert tokens.setdefault(n, got) == got
            assert sum(1 for key in session.graphs if len(key) > 3) <= 2


@pytest.mark.gpu
@pytest.mark.parametrize("rows", [0, 1 << 20], ids=["tcgen05", "streamed"])
def test_sums_stay_when_members_end(monkeypatch, rows):
    """Bit for bit: a member's next logits, whether its mates are still there or have ended (six sequences of two kv heads, so that
    the same warps take part)."""
    from mdma_b200.engine import Engine
    shared_whatever_the_size(monkeypatch, rows)
    d, c, _ = make_model(TINY_D, 2, torch.bfloat16, std_scale=SHARP)
    out = []
    for stay in (6, 2):
        eng = Engine(d, dtype="bfloat16", max_batch=6, max_context=2304)
        a = eng.acquire()
        step(eng, [(a, ids(TINY_D, 1021, 0))])
        slots = [a] + eng.fork(a, 5)
        got = [step(eng, [(s, [3 + i], [0]) for i, s in enumerate(slots)])]
        for s in slots[stay:]:
            eng.release(s)
        for turn in range(3):
            got.append(step(eng, [(s, [9 + turn], [0]) for s in slots[:stay]])[:2])
        out.append(got)
    assert all(np.array_equal(x[:2], y[:2]) for x, y in zip(*out))


@pytest.mark.gpu
@pytest.mark.parametrize("cfg, temperature", [(TINY_A, 0.0), (TINY_B, 0.0), (TINY_C, 0.9)], ids=["A", "B", "C"])
def test_completions_equal_those_of_repeated_prompts(cfg, temperature):
    from mdma_b200.engine import Engine
    d, c, tensors = make_model(cfg, 1, torch.float32, std_scale=SHARP)
    prompts = [ids(cfg, n, n) for n in (70, 16, 1)]
    eng = Engine(d, dtype="float32", max_batch=9, max_context=100, page_size=16)
    args = dict(max_tokens=14, temperature=temperature, seed=3, top_p=0.9)
    for graphs in (True, False):
        outs = eng.generate(prompts, n=3, use_graphs=graphs, **args)
        want = eng.generate([p for p in prompts for _ in range(3)], use_graphs=graphs, **args)
        assert [o.tokens for o in outs] == [o.tokens for o in want] and [o.prompt_tokens for o in outs] == [o.prompt_tokens for o in want]
        if temperature == 0.0:
            for p, o in zip(prompts, outs[::3]):
                assert o.tokens == plain_generate(c, tensors, p, 14)
        eng.cache.check()
        assert eng.cache.slots.free_count == 9 and all(g.pages.free_count == g.n_pages for g in eng.cache.groups)
    # more than fit at once, and a small cache
    small = Engine(d, dtype="float32", max_batch=4, max_context=100, page_size=16, max_tokens=16 * 9)
    outs = small.generate(prompts, n=3, **args)
    assert [o.tokens for o in outs] == [o.tokens for o in want]


@pytest.mark.gpu
def test_generation_takes_no_device_memory():
    from mdma_b200.engine import Engine
    d, _, _ = make_model(TINY_B, 1, torch.bfloat16, std_scale=SHARP)
    eng = Engine(d, max_batch=8, max_context=256)
    prompt = [ids(TINY_B, 100, 0)]
    eng.generate(prompt, max_tokens=20, n=8)
    torch.cuda.synchronize()
    before = torch.cuda.memory_allocated()
    for n in (8, 3, 1, 5):
        eng.generate(prompt, max_tokens=30, n=n, use_graphs=False, temperature=0.7)
    torch.cuda.synchronize()
    assert torch.cuda.memory_allocated() == before
    assert eng.held_bytes()["total_bytes"] == eng.memory_plan()["total_bytes"]


@pytest.mark.gpu
def test_command_line():
    d, _, _ = make_model(TINY_A, 0, torch.float32)
    run = lambda *a: subprocess.run([sys.executable, os.path.join(ROOT, "bin", "mdma"), "run", d, "5,17,3", "--json", "--dtype", "float32",  # noqa: E731
                                     "--max-tokens", "6", *a], capture_output=True, text=True, timeout=600)
    res = run("--n", "3")
    assert res.returncode == 0, res.stderr
    lines = [json.loads(line) for line in res.stdout.splitlines()]
    assert len(lines) == 3 and lines[0] == lines[1] == lines[2] and len(lines[0]["tokens"]) == 6
    assert run("--n", "0").returncode == 2
