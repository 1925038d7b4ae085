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
