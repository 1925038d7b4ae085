"""Which single-token steps read shared prefixes once, and what that is decided by."""
from types import SimpleNamespace

import pytest
import torch

from mdma_b200 import ops_tensor
from mdma_b200.cache import KVNeed, PrefixGroups, SequenceCache


def plan(families, lone, slots, context=16384, heads=32, kv_heads=8, page=64):
    """The plan of a step of families of (members, prefix) and of sequences alone, as an engine bounds it."""
    shared, pos0 = [], []
    for members, length in families:
        shared.append((length, list(range(len(pos0), len(pos0) + members))))
        pos0 += [length + 20] * members
    pos0 += [500] * lone
    g = PrefixGroups(shared, pos0, [1] * len(pos0))
    up = lambda n: min(context, -(-n // 1024) * 1024)  # noqa: E731
    g.most_len, g.most_own = up(g.most_len), up(g.most_own)
    ctx = SimpleNamespace(max_new=1, n_seqs=len(pos0), n_tokens=len(pos0), most_seqs=slots, most_len=context)
    return ops_tensor.prefix_plan(ctx, g, heads, kv_heads, 128, 148, page)


@pytest.mark.parametrize("families, lone, slots, alone", [([(2, 10)], 62, 64, True), ([(2, 500)], 62, 64, True), ([(16, 512)], 0, 64, True),
                                                         ([(64, 100)], 0, 64, True), ([(64, 1000)], 0, 64, False), ([(2, 2000)], 62, 64, False),
                                                         ([(8, 2000)], 0, 8, True), ([(8, 8000)], 0, 8, False), ([(20, 600), (20, 900)], 0, 64, False)])
def test_short_prefixes_of_few_are_read_by_every_sequence(families, lone, slots, alone):
    assert (plan(families, lone, slots)[0] == 0) == alone


def test_a_small_family_is_cut_for_itself_not_for_the_engine():
    assert plan([(2, 8000)], 0, 64)[0] >= 16 and plan([(2, 8000)], 62, 64)[0] >= 16
    assert plan([(2, 2000)], 0, 2)[0] == 0 and plan([(2, 16000)], 0, 2) == (32, 1, ops_tensor.PREFIX_STREAM)


def test_the_cache_remembers_what_families_shared():
    c = SequenceCache([KVNeed(2, 16)], [None], 64 * 40, 8, 1024, torch.float32, "cpu", 64, allocate=False)
    a = c.acquire()
    c.extend({a: 128})
    c.commit({a: 128})
    new = c.fork(a, 3, 70)
    b = c.acquire()
    assert c.shared_keys([a, b] + new) == 4 * 70 and c.shared_keys([b]) == 0
    c.release(new[0])
    assert c.shared_keys([a, new[1]]) == 4 * 70
    (d,) = c.fork(a)                                  # a's last fork counts; two are left of the first
    assert c.shared_keys([a, d] + new[1:]) == 2 * 128 + 4 * 70
    g = PrefixGroups([(70, [0, 2]), (128, [1])], [80, 200, 70, 9], [1] * 4)
    assert g.shared_keys == 2 * 70 + 128 and g.skips == [70, 128, 70, 0]


@pytest.mark.parametrize("members, length, new, kv_heads, page, pays", [
    (2, 64, 2, 8, 64, False), (4, 512, 3, 8, 64, False), (4, 1024, 3, 8, 64, True), (16, 256, 30, 32, 64, True), (2, 64, 20, 32, 64, False),
    (8, 512, 500, 8, 64, False), (24, 1024, 60, 8, 64, False), (64, 1024, 60, 8, 64, True), (24, 4100, 60, 8, 64, True), (2, 2048, 1000, 8, 64, True),
    (8, 2048, 500, 8, 16, False), (4, 2048, 3, 8, 16, True), (2, 64, 1, 8, 16, False), (4, 300, 1, 8, 16, True), (2, 4000, 1, 8, 16, True)])
def test_steps_that_gain_nothing_read_by_themselves(members, length, new, kv_heads, page, pays):
    g = PrefixGroups([(length, list(range(members)))], [length] * members, [new] * members)
    ctx = SimpleNamespace(max_new=new, n_seqs=members, n_tokens=new * members, most_seqs=64, most_len=16384)
    assert ops_tensor.prefix_pays(ctx, g, 32, kv_heads, 128, page) == pays
