"""A sequence's logits stay as they are, bit for bit, when members of its family end."""
import numpy as np
import pytest
import torch

from test_forks import ids, step
from tiny import SHARP, TINY_D, make_model


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
