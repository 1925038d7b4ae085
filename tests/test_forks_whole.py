"""A fork or a truncation that cannot be done leaves the cache as it was."""
import pytest
import torch

from mdma_b200.cache import KVNeed, SequenceCache, StateNeed
from mdma_b200.cache.kv import CacheGroup


def make(needs, states, device="cpu", allocate=True, tokens=64 * 12, slots=5):
    return SequenceCache(needs, states, tokens, slots, 512, torch.float32, device, 64, allocate=allocate)


def grow(c, slot, n):
    c.extend({slot: n})
    c.commit({slot: n})


def books(c):
    return (dict(c.lengths), dict(c.shares), dict(c.families), c.slots.free_count,
            [(g.pages.free_count, dict(g.holders), {s: dict(p) for s, p in g.seq_pages.items()}) for g in c.groups])


def test_state_off_the_gpu_does_not_fork():
    c = make([KVNeed(2, 16)], [StateNeed((3,))])
    a = c.acquire()
    grow(c, a, 64)                                   # (a whole page: no rows are to be copied)
    before = books(c)
    assert "GPU" in c.can_fork(a, 2)
    with pytest.raises(ValueError, match="GPU"):
        c.fork(a, 2)
    c.check()
    assert books(c) == before


@pytest.mark.parametrize("fails", ["pages", "state"])
def test_a_fork_whose_copies_fail_gives_everything_back(fails, monkeypatch):
    from mdma_b200 import ops
    c = make([KVNeed(2, 16), KVNeed(1, 8, window=100)], [StateNeed((3,)), None], allocate=False)
    a = c.acquire()
    grow(c, a, 150)
    (b,) = c.fork(a)
    c.states = {0: torch.zeros(5, 3)}
    monkeypatch.setattr(SequenceCache, "_fork_refusal", lambda *args: None)
    calls = []

    def copy(*args):
        calls.append(args)
        if fails == "pages" and len(calls) == 2:
            raise RuntimeError("no copy")
    monkeypatch.setattr(CacheGroup, "copy", copy)

    def copy_slots(*args):
        raise RuntimeError("no copy")
    monkeypatch.setattr(ops, "copy_slots", copy_slots)
    monkeypatch.setattr(torch.cuda, "device", lambda d: pytest.MonkeyPatch.context())
    before = books(c)
    with pytest.raises(RuntimeError, match="no copy"):
        c.fork(a, 2)
    c.check()
    assert books(c) == before and len(calls) == 2
    c.release(a)
    c.release(b)
    c.check()
    assert all(g.pages.free_count == g.n_pages for g in c.groups)


@pytest.mark.parametrize("free", [0, 3])
def test_a_truncation_whose_copy_fails_changes_nothing(free, monkeypatch):
    c = make([KVNeed(2, 16), KVNeed(1, 8)], [None, None], allocate=False, tokens=64 * (5 + free))
    a = c.acquire()
    grow(c, a, 192)
    (b,) = c.fork(a)
    grow(c, b, 100)                                  # two pages of its own behind the shared ones
    calls = []

    def copy(*args):
        calls.append(args)
        if len(calls) == 2:
            raise RuntimeError("no copy")
    monkeypatch.setattr(CacheGroup, "copy", copy)
    before = books(c)
    with pytest.raises(RuntimeError, match="no copy"):
        c.truncate(b, 100)
    c.check()
    assert books(c) == before
    calls.clear()
    calls.append(None)
    monkeypatch.setattr(CacheGroup, "copy", lambda *args: calls.append(args))
    c.truncate(b, 100)
    c.check()
    for (group, src, dst, rows), g in zip(calls[1:], c.groups):
        assert group is g and src == [g.seq_pages[a][1]] and dst == [g.seq_pages[b][1]] and rows == [36] and src != dst
    assert len(calls) == 3 and c.length(b) == 100 and all(sorted(g.seq_pages[b]) == [0, 1] for g in c.groups)


@pytest.mark.parametrize("after", [0, 1, 3])
def test_cancelled_completions_say_so(after):
    """Cancelled before the prompt, or after some tokens: every completion ends with that reason and no slot stays held."""
    from mdma_b200.engine.generate import FINISH_CANCELLED, Generator
    from test_forks import FakeEngine, FakeSampler
    engine, asked = FakeEngine(8, 100), []

    def cancelled():
        asked.append(1)
        return len(asked) > after
    outs = Generator(engine, FakeSampler(), use_graphs=False).generate([[1, 2, 3], [4]], 9, n=3, cancelled=cancelled)
    assert [o.finish_reason for o in outs] == [FINISH_CANCELLED] * 6 and not engine.live
    assert all(len(o.tokens) == after for o in outs)
