"""Compaction where there is something to move: holes in front of held pages, some of which several sequences hold."""
import numpy as np
import pytest
import torch

from plain_llama import plain_forward
from replay_util import assert_close
from test_cache_pages import grow, make
from test_forks import ids, step
from tiny import SHARP, TINY_A, make_model
from mdma_b200.cache import KVNeed


def test_shared_pages_move_for_all_their_holders():
    c = make([KVNeed(2, 16), KVNeed(1, 8, window=100)])
    gone, a = c.acquire(), c.acquire()
    grow(c, gone, 400)
    grow(c, a, 150)
    b, d = c.fork(a, 2)
    grow(c, b, 100)
    c.release(gone)
    before = {s: dict(c.groups[0].seq_pages[s]) for s in (a, b, d)}
    moved = c.compact()
    c.check()
    g = c.groups[0]
    assert moved > 0 and max(g.pages.held) == len(g.pages.held) - 1
    assert g.seq_pages[a][0] == g.seq_pages[b][0] == g.seq_pages[d][0] != before[a][0] and g.holders[g.seq_pages[a][0]] == 3
    for s in (a, b, d):
        assert all(g.table_host[s, p] == page for p, page in g.seq_pages[s].items())
    assert c.compact() == 0


@pytest.mark.gpu
def test_rows_follow_their_pages():
    c = make([KVNeed(2, 16), KVNeed(3, 8, values=False), KVNeed(1, 4, v_dim=12)], device="cuda")
    gone, a = c.acquire(), c.acquire()
    grow(c, gone, 400)
    grow(c, a, 150)
    b, d = c.fork(a, 2)
    for g in c.groups:
        for t in (g.k, g.v):
            if t is not None:
                t.normal_()

    def rows():
        return [t[:, g.table_dev[s].long()].flatten(1, 2)[:, :150].clone() for g in c.groups for t in (g.k, g.v) if t is not None for s in (a, b, d)]
    want = rows()
    c.release(gone)
    assert c.compact() == 5 * len(c.groups)          # (all of them: seven pages lay in front)
    c.check()
    assert all(max(g.pages.held) == len(g.pages.held) - 1 for g in c.groups)
    c.poison_unused()
    assert all(torch.equal(x, y) for x, y in zip(rows(), want))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
def test_steps_after_pages_moved(dtype):
    from mdma_b200.engine import Engine
    d, c, tensors = make_model(TINY_A, 1, torch.bfloat16, std_scale=SHARP)
    weights = {k: v.float() for k, v in tensors.items()}
    eng = Engine(d, dtype=dtype, max_batch=6, max_context=128, page_size=16, logit_rows=16)
    gone, a = eng.acquire(), eng.acquire()
    text = ids(TINY_A, 75, 0)
    step(eng, [(gone, ids(TINY_A, 90, 1)), (a, text)])
    slots = [a] + eng.fork(a, 3)
    session = eng.decode_session()
    session.start(slots, [5, 6, 7, 8])
    session.run(1)
    session.read()
    eng.release(gone)
    assert eng.compact() > 0
    eng.cache.poison_unused()
    eng.cache.check()
    got = step(eng, [(s, [9, 10 + i], [0, 1]) for i, s in enumerate(slots)])
    want = [plain_forward(c, weights, text + [5 + i, 9, 10 + i], torch.float64).numpy()[-2:] for i in range(4)]
    assert_close(got, np.concatenate(want), dtype, "moved")
