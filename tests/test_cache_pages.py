"""Pages of the cache that several sequences hold: forks, frees, truncation, compaction; and the kernel that copies pages."""
import random

import pytest
import torch

from mdma_b200 import ops
from mdma_b200.cache import CacheFull, KVNeed, SequenceCache, StateNeed
from mdma_b200.ops import KernelError


def make(needs=(KVNeed(2, 16),), states=None, tokens=64 * 40, slots=8, ctx=1024, page=64, device=None):
    states = list(states) if states is not None else [None] * len(needs)
    if device is None:
        return SequenceCache(list(needs), states, tokens, slots, ctx, torch.float32, "cpu", page, allocate=False)
    return SequenceCache(list(needs), states, tokens, slots, ctx, torch.float32, device, page)


def grow(c, slot, n):
    c.extend({slot: n})
    c.commit({slot: n})


# ---- bookkeeping, on the CPU ----------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("length, full, part", [(0, 0, 0), (1, 0, 1), (63, 0, 1), (64, 1, 0), (65, 1, 1), (200, 3, 1)])
def test_a_fork_shares_full_pages_and_copies_the_last_one(length, full, part):
    c = make()
    a = c.acquire()
    if length:
        grow(c, a, length)
    g = c.groups[0]
    used = g.n_pages - g.pages.free_count
    new = c.fork(a, 3)
    c.check()
    assert len(new) == 3 and all(c.length(s) == length for s in new)
    assert g.n_pages - g.pages.free_count == used + 3 * part
    for s in new:
        assert [g.seq_pages.get(s, {}).get(p) for p in range(full)] == [g.seq_pages[a][p] for p in range(full)] if full else True
        if part:
            assert g.seq_pages[s][full] != g.seq_pages[a][full]
        assert g.table_host[s, :full].tolist() == g.table_host[a, :full].tolist()
    for s in [a] + new[:2]:
        c.release(s)
        c.check()
    assert c.length(new[2]) == length and g.n_pages - g.pages.free_count == full + part
    c.release(new[2])
    c.check()
    assert g.pages.free_count == g.n_pages and not g.holders and not c.shares


def test_fork_at_an_earlier_length():
    c = make()
    a = c.acquire()
    grow(c, a, 300)
    (b,) = c.fork(a, 1, 130)
    assert c.length(b) == 130 and sorted(c.groups[0].seq_pages[b]) == [0, 1, 2]
    c.check()
    assert c.shared_prefixes([b, a]) == [(130, [0, 1])]


def test_forks_are_refused_whole():
    c = make(tokens=64 * 5, slots=4)
    a = c.acquire()
    grow(c, a, 200)                                   # four pages, one is free
    before = (c.slots.free_count, c.groups[0].pages.free_count)
    for n, length, error in [(2, None, CacheFull), (4, 192, CacheFull), (0, None, ValueError), (1, 201, ValueError), (1, -1, ValueError)]:
        with pytest.raises(error):
            c.fork(a, n, length)
        assert (c.slots.free_count, c.groups[0].pages.free_count) == before
        assert c.can_fork(a, n, length)
    with pytest.raises(ValueError):
        c.fork(a + 1)
    c.check()
    assert c.can_fork(a, 3, 192) is None and len(c.fork(a, 3, 192)) == 3
    c.check()


def test_windowed_groups_share_what_is_left():
    c = make([KVNeed(2, 16), KVNeed(2, 16, window=100), KVNeed(2, 16, window=70, keep_first=3), KVNeed(2, 16, chunk=100)])
    a = c.acquire()
    for n in (400, 50, 3):
        grow(c, a, n)
    new = c.fork(a, 2)
    c.check()
    with pytest.raises(ValueError, match="released"):
        c.fork(a, 1, 200)
    for n in (1, 90, 200):
        for s in [a] + new:
            grow(c, s, n)
            c.check()
    for s in new + [a]:
        c.release(s)
        c.check()
    assert all(g.pages.free_count == g.n_pages for g in c.groups)


def test_state_forks_at_the_end_only():
    c = make([KVNeed(2, 16)], [StateNeed((4,))])
    a = c.acquire()
    grow(c, a, 10)
    with pytest.raises(ValueError, match="end only"):
        c.fork(a, 1, 9)


def test_truncation_into_a_shared_page_copies_it():
    c = make(tokens=64 * 6)
    a = c.acquire()
    grow(c, a, 192)
    (b,) = c.fork(a)
    g = c.groups[0]
    c.truncate(b, 128)                                # ends with a full page: nothing to copy
    assert g.seq_pages[b][1] == g.seq_pages[a][1] and c.shared_prefixes([a, b]) == [(192, [0])]
    c.truncate(b, 100)
    assert g.seq_pages[b][1] != g.seq_pages[a][1] and g.seq_pages[b][0] == g.seq_pages[a][0]
    c.check()
    d = c.acquire()
    grow(c, d, 128)                                   # the last two pages
    (e,) = c.fork(a)
    with pytest.raises(CacheFull):
        c.truncate(e, 100)
    c.check()
    assert c.length(e) == 192


def test_the_last_fork_counts():
    c = make()
    a = c.acquire()
    grow(c, a, 70)
    b, d = c.fork(a, 2)
    grow(c, b, 30)
    (e,) = c.fork(b)
    assert c.shared_prefixes([a, b, d, e]) == [(70, [0, 2]), (100, [1, 3])]
    (f,) = c.fork(a)
    assert c.shared_prefixes([a, d, f]) == [(70, [0, 1, 2])]
    for s in (a, b, d, e, f):
        c.release(s)
    assert c.shared_prefixes([]) == [] and not c.shares


def test_families_are_remembered_while_someone_is_left():
    c = make()
    a = c.acquire()
    grow(c, a, 70)
    b, d = c.fork(a, 2)
    assert c.most_members([a, b, d]) == 3 and c.most_members([]) == 0
    c.release(b)
    c.release(d)
    assert c.most_members([a]) == 3                   # who has ended counts on
    for _ in range(5):                                # one after the other, never more than three at a time
        (e,) = c.fork(a)
        c.release(e)
    assert c.most_members([a]) == 3 and len(c.families) == 1
    grow(c, a, 30)
    (e,) = c.fork(a)                                  # another fork: nobody is left of the first
    assert c.most_members([a, e]) == 2 and len(c.families) == 1
    c.truncate(e, 64)
    assert c.most_members([e]) == 0 and c.most_members([a]) == 2
    c.release(a)
    c.release(e)
    assert not c.families and not c.shares


def test_random_traffic_with_forks_loses_nothing():
    rng = random.Random(5)
    c = make([KVNeed(2, 16), KVNeed(1, 32, window=100)], tokens=64 * 30, slots=9, ctx=700)
    live = {}
    for _ in range(1500):
        what = rng.random()
        if live and what < 0.2:
            slot = rng.choice(list(live))
            c.release(slot)
            del live[slot]
        elif what < 0.3 and c.slots.free_count:
            live[c.acquire()] = 0
        elif live and what < 0.5:
            slot, n = rng.choice(list(live)), rng.randint(1, 3)
            if c.can_fork(slot, n) is None:
                for s in c.fork(slot, n):
                    live[s] = live[slot]
        elif what < 0.55:
            c.compact()
            assert all(max(g.pages.held, default=-1) == len(g.pages.held) - 1 for g in c.groups)
        elif live:
            ext = {s: rng.randint(1, 90) for s in rng.sample(list(live), rng.randint(1, len(live)))}
            if c.can_extend(ext) is None:
                c.extend(ext)
                c.commit(ext)
                for s, n in ext.items():
                    live[s] += n
        c.check()
        for s, n in live.items():
            assert c.length(s) == n
            have = c.groups[0].seq_pages.get(s, {})
            assert sorted(have) == list(range(-(-n // 64))) and [c.groups[0].table_host[s, p] for p in sorted(have)] == [have[p] for p in sorted(have)]
    for s in list(live):
        c.release(s)
    c.check()
    assert all(g.pages.free_count == g.n_pages and not g.holders for g in c.groups)


def test_copies_need_the_gpu():
    with pytest.raises(KernelError, match="no CPU path"):
        ops.copy_pages([torch.zeros(1, 4, 8, 2)], [0], [1])


# ---- the kernel -----------------------------------------------------------------------------------------------------------------
def pool(shape, dtype, seed):
    gen = torch.Generator().manual_seed(seed)
    t = torch.randint(0, 256, (*shape, torch.empty((), dtype=dtype).element_size()), generator=gen, dtype=torch.uint8)
    return t.view(dtype).reshape(shape)


def expect(before, src, dst, rows):
    out = before.clone()
    for i, (a, b) in enumerate(zip(src, dst)):
        n = before.shape[2] if rows is None else rows[i]
        out[:, b, :n] = before[:, a, :n]
    return out


def same(a, b):
    raw = lambda t: torch.empty(t.shape, dtype=t.dtype).copy_(t).flatten().view(torch.uint8)  # noqa: E731
    return torch.equal(raw(a), raw(b))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.uint8], ids=str)
@pytest.mark.parametrize("shape", [(1, 12, 64, 2, 16), (3, 12, 16, 1, 5), (2, 12, 7, 3, 3), (5, 12, 1, 1, 1), (2, 12, 128, 8, 128), (33, 12, 2, 1, 24)], ids=str)
def test_copies_equal_indexing(shape, dtype):
    ps = shape[2]
    cases = [([0], [1], None), ([3] * 5 + [9], [0, 1, 2, 4, 5, 11], None), ([11, 2, 2, 7], [0, 1, 3, 10], [ps, 1, 0, max(1, ps // 2)]),
             ([4] * 7, [0, 1, 2, 3, 5, 6, 7], [max(1, ps - 1)] * 7), ([], [], None)]
    for src, dst, rows in cases:
        a, b = pool(shape, dtype, 1), pool((shape[0] + 1, *shape[1:3], 3), dtype, 2)
        on = [a.cuda(), b.cuda()]
        ops.copy_pages(on, src, dst, rows)
        assert same(on[0].cpu(), expect(a, src, dst, rows)) and same(on[1].cpu(), expect(b, src, dst, rows))


@pytest.mark.gpu
def test_many_copies_and_many_pools():
    gen = random.Random(3)
    pages = 5000
    order = list(range(pages))
    gen.shuffle(order)
    src, dst = [order[gen.randrange(900)] for _ in range(3300)], order[1000:4300]
    rows = [gen.randint(0, 4) for _ in src]
    pools = [pool((1 + i % 2, pages, 4, 1 + i % 3), torch.float32, i) for i in range(40)]
    on = [p.cuda() for p in pools]
    before = ops.LAUNCHES
    ops.copy_pages(on, src, dst, rows)
    assert ops.LAUNCHES > before
    for p, q in zip(pools, on):
        want = p.clone()
        for r in range(4):
            pick = [i for i in range(len(src)) if rows[i] > r]
            want[:, [dst[i] for i in pick], r] = p[:, [src[i] for i in pick], r]
        assert same(q.cpu(), want)


@pytest.mark.gpu
def test_copies_into_a_view_of_wider_memory():
    whole = torch.arange(4 * 6 * 8 * 3, dtype=torch.float32, device="cuda")
    p = whole[3:3 + 2 * 6 * 8 * 3].view(2, 6, 8, 3)          # an address that only floats are aligned to
    want = expect(p.cpu(), [5, 5], [0, 2], [8, 8])
    rest = whole[3 + p.numel():].clone()
    ops.copy_pages([p], [5, 5], [0, 2], [8, 8])
    assert torch.equal(p.cpu(), want) and torch.equal(rest, whole[3 + p.numel():])


def test_a_cache_off_the_gpu_does_not_fork_inside_a_page():
    c = SequenceCache([KVNeed(2, 16)], [None], 64 * 8, 4, 256, torch.float32, "cpu", 64)
    a = c.acquire()
    grow(c, a, 70)
    with pytest.raises(ValueError, match="GPU"):
        c.fork(a)
    c.check()
    (b,) = c.fork(a, 1, 64)
    with pytest.raises(ValueError, match="GPU"):
        c.truncate(b, 10)
    c.check()
    assert c.length(a) == 70 and c.length(b) == 64


@pytest.mark.gpu
def test_pools_of_nothing_and_pages_of_one_row():
    a, b = pool((2, 6, 1, 3), torch.float32, 0), pool((1, 6, 1, 1), torch.bfloat16, 1)
    on = [torch.empty(0, 6, 1, 4, device="cuda"), a.cuda(), torch.empty(2, 6, 1, 0, device="cuda"), b.cuda().as_strided((1, 6, 1, 1), (99, 1, 77, 5))]
    ops.copy_pages(on, [2, 2, 5], [0, 1, 3], [1, 0, 1])
    want = [expect(x, [2, 5], [0, 3], None) for x in (a, b)]
    assert same(on[1].cpu(), want[0]) and same(on[3].cpu(), want[1])
    ops.copy_pages(on[:1], [2], [0])


@pytest.mark.gpu
def test_copies_refuse_and_leave_the_pools():
    p = pool((2, 6, 8, 3), torch.float32, 0).cuda()
    before = p.clone()
    for src, dst, rows in [([0], [6], None), ([-1], [2], None), ([0, 1], [2, 2], None), ([0, 2], [2, 3], None), ([0], [0], None),
                           ([0], [1], [9]), ([0], [1], [-1]), ([0, 1], [2], None), ([0], [1], [])]:
        with pytest.raises(KernelError):
            ops.copy_pages([p], src, dst, rows)
    with pytest.raises(KernelError):
        ops.copy_pages([p, p[:, :5].contiguous()], [0], [1])
    with pytest.raises(KernelError):
        ops.copy_pages([p.transpose(0, 1)], [0], [1])
    for src in ([2 ** 40], [0.5], ["a"]):
        with pytest.raises(KernelError):
            ops.copy_pages([p], src, [1])
    assert same(p, before)
    ops.copy_pages([], [0], [1])


@pytest.mark.gpu
def test_a_captured_copy_keeps_its_list():
    p = pool((2, 6, 8, 4), torch.bfloat16, 0).cuda()
    src, dst = [0, 0], [1, 2]
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        ops.copy_pages([p], src, dst)
    src[0], dst[0] = 4, 5
    q = pool((2, 6, 8, 4), torch.bfloat16, 9).cuda()
    p.copy_(q)
    graph.replay()
    assert same(p.cpu(), expect(q.cpu(), [0, 0], [1, 2], None))


@pytest.mark.gpu
def test_forked_caches_hold_the_same_rows():
    c = make([KVNeed(2, 16), KVNeed(3, 8, values=False), KVNeed(1, 4, v_dim=12)], [StateNeed((5, 3)), None, StateNeed((7,), torch.float64)], device="cuda")
    a = c.acquire()
    grow(c, a, 150)
    for g in c.groups:
        for t in (g.k, g.v):
            if t is not None:
                t.normal_()
    for s in c.states.values():
        s.normal_()

    def rows(slot, n):
        out = []
        for g in c.groups:
            table = g.table_dev[slot].long()
            for t in (g.k, g.v):
                if t is not None:
                    out.append(t[:, table].flatten(1, 2)[:, :n])
        return out
    want = [t.clone() for t in rows(a, 150)]
    state = {i: s[a].clone() for i, s in c.states.items()}
    new = c.fork(a, 4)
    for s in new:
        assert all(torch.equal(x, y) for x, y in zip(rows(s, 150), want))
        assert all(torch.equal(t[s], state[i]) for i, t in c.states.items())
    c.poison_unused()
    c.release(a)
    c.release(new[1])
    c.poison_unused()
    moved = c.compact()
    c.poison_unused()
    c.check()
    assert moved >= 0 and all(max(g.pages.held) == len(g.pages.held) - 1 for g in c.groups)
    for s in (new[0], new[2], new[3]):
        assert all(torch.equal(x, y) for x, y in zip(rows(s, 150), want))
