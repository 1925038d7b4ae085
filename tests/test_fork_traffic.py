"""Random traffic with forks: prompts, forks at any length, truncations, ends, moved pages, steps of one token and of several, replayed
steps; every logit row against the plain implementation, every row that nobody owns holds NaN."""
import random

import numpy as np
import pytest
import torch

from plain_llama import plain_forward
from replay_util import assert_close
from test_forks import ids, shared_whatever_the_size
from tiny import SHARP, TINY_A, TINY_B, TINY_D, make_model


@pytest.mark.gpu
@pytest.mark.parametrize("how", ["as it pays", "tcgen05", "streamed"])
@pytest.mark.parametrize("cfg, page", [(TINY_A, 16), (TINY_B, 64), (TINY_D, 32)], ids=["A-16", "B-64", "D-32"])
@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
def test_traffic(dtype, cfg, page, how, monkeypatch):
    from mdma_b200.engine import Engine, StepEntry
    if how != "as it pays":
        if dtype == "float32":
            pytest.skip("one way only")
        shared_whatever_the_size(monkeypatch, 0 if how == "tcgen05" else 1 << 20)
    d, c, tensors = make_model(cfg, 1, torch.bfloat16, std_scale=SHARP)
    weights = {k: v.float() for k, v in tensors.items()}
    eng = Engine(d, dtype=dtype, max_batch=9, max_context=128, page_size=page, max_tokens=None, logit_rows=32)
    rng, text, shared_steps = random.Random(page), {}, 0

    def check(got, rows, what):
        nonlocal shared_steps
        assert_close(np.stack(got), np.stack([plain_forward(c, weights, t, torch.float64).numpy()[-1] for t in rows]), dtype, what)
    for turn in range(70):
        what = rng.random()
        room = {s: 127 - len(t) for s, t in text.items()}
        if len(text) < 3 or (what < 0.12 and eng.cache.slots.free_count):
            if eng.cache.slots.free_count:
                s = eng.acquire()
                text[s] = ids(cfg, rng.randint(1, 70), turn)
                check(eng.step([StepEntry(s, text[s], [len(text[s]) - 1])]).double().cpu().numpy(), [text[s]], f"turn {turn}: a prompt")
        elif what < 0.34:
            s = rng.choice(list(text))
            n = rng.randint(1, 3)
            length = len(text[s]) if rng.random() < 0.6 else rng.randint(0, len(text[s]))
            if eng.cache.can_fork(s, n, length) is None:
                for new in eng.fork(s, n, length):
                    text[new] = text[s][:length]
        elif what < 0.44:
            s = rng.choice(list(text))
            length = rng.randint(0, len(text[s]))
            eng.cache.truncate(s, length)
            text[s] = text[s][:length]
        elif what < 0.54:
            s = rng.choice(list(text))
            eng.release(s)
            del text[s]
        elif what < 0.6:
            eng.compact()
        elif what < 0.72:
            some = [s for s in text if room[s] > 9]
            if some:
                news = {s: ids(cfg, rng.randint(1, 9), 1000 * turn + s) for s in rng.sample(some, rng.randint(1, len(some)))}
                if eng.cache.can_extend({s: len(t) for s, t in news.items()}) is None:
                    got = eng.step([StepEntry(s, t, [len(t) - 1]) for s, t in news.items()]).double().cpu().numpy()
                    eng.check_status()
                    for s, t in news.items():
                        text[s] = text[s] + t
                    check(got, [text[s] for s in news], f"turn {turn}: several tokens")
        else:
            some = [s for s in text if room[s] > 2 and text[s]]
            some = rng.sample(some, rng.randint(min(2, len(some)), len(some))) if some else []
            if some and eng.cache.can_extend({s: 1 for s in some}) is None:
                shared_steps += eng.prefix_groups(some, [eng.cache.length(s) for s in some], [1] * len(some)) is not None
                tokens = [rng.randrange(cfg["vocab_size"]) for _ in some]
                if rng.random() < 0.5:
                    got = eng.step([StepEntry(s, [t], [0]) for s, t in zip(some, tokens)]).double().cpu().numpy()
                else:
                    session = eng.decode_session()
                    session.start(some, tokens)
                    session.run(1)
                    session.read()
                    got = session.logits[:len(some)].double().cpu().numpy()
                eng.check_status()
                for s, t in zip(some, tokens):
                    text[s] = text[s] + [t]
                check(got, [text[s] for s in some], f"turn {turn}: one token each")
        eng.cache.poison_unused()
        eng.cache.check()
        assert {s: len(t) for s, t in text.items()} == eng.cache.lengths
    assert shared_steps > 3 or (dtype == "bfloat16" and how == "as it pays")
