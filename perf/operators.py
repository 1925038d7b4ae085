"""The operators of batches that share their beginning: pages of the cache copied for forks and moves, and attention whose
shared prefix is read once for all of its sequences.

`listed()` are the measured cases, `draw(rng)` more of the same ranges.  `run(state)` makes one pass: the plain form in
elementary torch operations, or, where `own` is set, the calls a user makes of the framework.  Head and layer sizes are those
of the configurations in `bench.py` and of the tests.

Copies (`op` "fork" and "move").  The pools hold [sites, pages, page_size, heads, dim] for keys and values.  A fork gives every
child of a parent its own copy of the parent's last, partly filled page: `rows` leading rows of it at every site.  A move
brings whole pages from the rear of the pool to free ones at its front.

Attention (`op` "decode" and "prompts").  Groups of sequences share their first tokens (the pages that these fill are the same
in their page tables; the last, partly filled one is a copy each); every sequence goes on with tokens of its own.  A step
brings one token a sequence, or several.  q rows are those of the fused projection [q heads | k heads | v heads], so they
lie further apart than the queries are wide."""
import math
from types import SimpleNamespace

import torch

own = False

DTYPES = {"bfloat16": torch.bfloat16, "float32": torch.float32}


# ---- cases ------------------------------------------------------------------------------------------------------------------
def _copies(name, op, dtype, sites, pages, page_size, kv_heads, dim, parents, children, rows):
    c = dict(op=op, dtype=dtype, sites=sites, pages=pages, page_size=page_size, kv_heads=kv_heads, dim=dim, parents=parents,
             children=children, rows=rows)
    return c if name is None else dict(c, name=name)


def _attention(name, op, dtype, heads, kv_heads, dim, page_size, groups, members, alone, prefix, before, new, sink=False):
    c = dict(op=op, dtype=dtype, heads=heads, kv_heads=kv_heads, dim=dim, page_size=page_size, groups=groups, members=members,
             alone=alone, prefix=prefix, before=before, new=new, sink=sink)
    return c if name is None else dict(c, name=name)


def listed():
    return [
        # the smallest call: one prompt of a small model goes on in four ways
        _copies("fork_1b_into_4", "fork", "bfloat16", 16, 64, 64, 8, 64, 1, 3, 37),
        # many samples of one prompt at the 8B shape
        _copies("fork_8b_into_64", "fork", "bfloat16", 32, 160, 64, 8, 128, 1, 63, 41),
        # sequences left the cache: the pages that are held move to its front
        _copies("move_1b_512_pages", "move", "bfloat16", 16, 1056, 64, 8, 64, 512, 1, 64),
        # the 32-bit engine: short pages, heads of an odd size, several prompts fork at once
        _copies("fork_float32_odd", "fork", "float32", 3, 96, 16, 2, 36, 5, 7, 11),
        # the smallest step: four samples of one short prompt, a small model
        _attention("decode_1b_4", "decode", "bfloat16", 32, 8, 64, 64, 1, 4, 0, 300, 23, 1),
        # an ordinary step: sixteen samples of one prompt
        _attention("decode_8b_16", "decode", "bfloat16", 32, 8, 128, 64, 1, 16, 0, 2048, 511, 1),
        # the largest: a long document in front of 64 users' sequences
        _attention("decode_8b_64_long", "decode", "bfloat16", 32, 8, 128, 64, 1, 64, 0, 32717, 900, 1),
        # several prompts with several samples each, sequences that share nothing among them; a key head per query head
        _attention("decode_7b_groups", "decode", "bfloat16", 32, 32, 128, 64, 6, 8, 3, 1500, 200, 1, sink=True),
        # short questions of unequal lengths behind one document
        _attention("prompts_8b_questions", "prompts", "bfloat16", 32, 8, 128, 64, 1, 24, 0, 4100, 0, 60),
        # longer prompts behind one document, some with turns before
        _attention("prompts_8b_long", "prompts", "bfloat16", 32, 8, 128, 64, 1, 8, 1, 8003, 130, 512),
        # the exact engine: eight samples of one prompt, a sink in the softmax
        _attention("decode_float32_8", "decode", "float32", 32, 8, 128, 64, 1, 8, 0, 1000, 60, 1, sink=True),
        # the exact engine: short pages, heads of an odd size, three groups and one sequence alone
        _attention("prompts_float32_odd", "prompts", "float32", 16, 2, 80, 16, 3, 3, 1, 500, 20, 40),
    ]


def _spread(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    if rng.random() < 0.35:
        dtype = rng.choice(["bfloat16", "bfloat16", "float32"])
        sites, page_size = rng.choice([1, 3, 4, 16, 32]), rng.choice([16, 32, 64, 64, 128])
        kv_heads, dim = rng.choice([1, 2, 8, 8, 32]), rng.choice([20, 36, 64, 80, 128, 128])
        page = sites * page_size * kv_heads * dim * 2 * (2 if dtype == "bfloat16" else 4)      # keys and values
        most = max(8, min(2000, 1_400_000_000 // page))                 # pages in the pool
        if rng.random() < 0.5:
            moved = _spread(rng, 1, most * 2 // 5)
            return _copies(None, "move", dtype, sites, min(most, 2 * moved + rng.randint(2, 40)), page_size, kv_heads, dim, moved, 1, page_size)
        parents = rng.randint(1, 6)
        children = _spread(rng, 1, max(1, min(64, (most - parents) // parents - 1)))
        return _copies(None, "fork", dtype, sites, min(most, parents * (children + 1) + rng.randint(1, 40)), page_size, kv_heads, dim, parents,
                       children, rng.randint(1, page_size))
    dtype = rng.choice(["bfloat16", "bfloat16", "bfloat16", "float32"])
    heads, kv_heads, dim = rng.choice([(32, 8, 128), (32, 8, 128), (32, 8, 64), (32, 32, 128), (12, 4, 80), (16, 2, 128), (20, 4, 64), (8, 1, 96)])
    page_size = rng.choice([16, 32, 64, 64, 64, 128])
    groups, alone = rng.choice([1, 1, 1, 2, 5]), rng.choice([0, 0, 1, 4])
    decode, wide = rng.random() < 0.6, dtype == "bfloat16"
    members = max(1, _spread(rng, 2, (96 if wide else 16) if decode else (32 if wide else 8)) // groups)
    n = groups * members + alone
    prefix = _spread(rng, 20, min(32000, (2_000_000 if wide else 40_000) // n * 1024 // max(1024, kv_heads * dim)))
    before = rng.choice([0, _spread(rng, 1, 1000 if wide else 100)])
    new = 1 if decode else _spread(rng, 2, max(3, min(500, (4_000_000 if wide else 200_000) // (n * (prefix + before)) + 3)))
    return _attention(None, "decode" if decode else "prompts", dtype, heads, kv_heads, dim, page_size, groups, members, alone, prefix,
                      before, new, sink=rng.random() < 0.3)


# ---- sizes ------------------------------------------------------------------------------------------------------------------
def _pairs(case):
    """(page to copy from, page to copy to, leading rows) of every copy."""
    n, pages = case["parents"], case["pages"]
    if case["op"] == "move":
        src = [pages - 1 - (i * 7 + 3) % n if math.gcd(7, n) == 1 else pages - 1 - i for i in range(n)]
        return src, list(range(n)), [case["rows"]] * n
    src, dst, rows = [], [], []
    for i in range(n):
        for j in range(case["children"]):
            src.append(pages - 1 - i)
            dst.append(i + j * n)
            rows.append(1 + (case["rows"] - 1 + 5 * i) % case["page_size"])
    return src, dst, rows


def _sequences(case):
    """(group or -1, tokens shared, own tokens before the step, new tokens) of every sequence, the groups' members in turn."""
    n_groups, out = case["groups"], []
    n = n_groups * case["members"] + case["alone"]
    for i in range(n):
        share = (i * 5 + 2) % n / max(1, n - 1)                       # from 0 to 1 over the sequences, in no order
        before = int(round(case["before"] * share))
        new = 1 if case["op"] == "decode" else max(1, int(round(case["new"] * (1.0 - 0.9 * share))))
        g = i % n_groups if i < n_groups * case["members"] else -1
        prefix = max(1, case["prefix"] - g * case["prefix"] // (2 * n_groups)) if g >= 0 else 0
        out.append((g, prefix, before, new))
    return out


# ---- a user's program ---------------------------------------------------------------------------------------------------------
def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(int(seed) * 7919 + 17)
    dtype = DTYPES[case["dtype"]]
    normal = lambda *shape: torch.randn(shape, generator=gen, device="cuda", dtype=torch.float32).to(dtype)  # noqa: E731
    s = SimpleNamespace(case=dict(case))
    if case["op"] in ("fork", "move"):
        shape = (case["sites"], case["pages"], case["page_size"], case["kv_heads"], case["dim"])
        s.k, s.v = normal(*shape), normal(*shape)
        s.src, s.dst, s.rows = _pairs(case)
        s.src_dev, s.dst_dev, s.rows_dev = (torch.tensor(x, device="cuda") for x in (s.src, s.dst, s.rows))
        return s
    seqs, ps = _sequences(case), case["page_size"]
    host = torch.Generator().manual_seed(int(seed) * 104729 + 5)
    # page tables: whole pages of a prefix are shared, everything behind them is a sequence's own
    whole = {g: prefix // ps for g, prefix, _, _ in seqs if g >= 0}
    lengths = [prefix + before + new for _, prefix, before, new in seqs]
    max_pages = max(-(-n // ps) for n in lengths)
    n_pages = sum(whole.values()) + sum(-(-n // ps) - whole.get(q[0], 0) for n, q in zip(lengths, seqs))
    order, at = torch.randperm(n_pages, generator=host), 0
    shared = {}
    for g, n in whole.items():
        shared[g] = order[at:at + n]
        at += n
    n_slots = len(seqs) + 2
    slots = torch.randperm(n_slots, generator=host)[:len(seqs)]
    table = torch.zeros(n_slots, max_pages, dtype=torch.int32)
    for slot, n, q in zip(slots, lengths, seqs):
        first, last = whole.get(q[0], 0), -(-n // ps)
        table[slot, :first] = shared.get(q[0], order[:0]).int()
        table[slot, first:last] = order[at:at + last - first].int()
        at += last - first
    s.k, s.v = (normal(n_pages, ps, case["kv_heads"], case["dim"]) for _ in range(2))
    # the partly filled last page of a prefix: every member's copy holds the same rows
    for g, n in whole.items():
        of = [i for i, q in enumerate(seqs) if q[0] == g]
        part = seqs[of[0]][1] - n * ps
        if part and len(of) > 1:
            first, rest = int(table[slots[of[0]], n]), table[slots[of[1:]], n].long().cuda()
            for pool in (s.k, s.v):
                pool[rest, :part] = pool[first, :part]
    news = [q[3] for q in seqs]
    ints = lambda x: torch.tensor(x, dtype=torch.int32, device="cuda")  # noqa: E731
    starts = [0]
    for n in news:
        starts.append(starts[-1] + n)
    pos0 = [q[1] + q[2] for q in seqs]
    s.n_seqs, s.n_tokens, s.max_new, s.max_len = len(seqs), starts[-1], max(news), max(lengths)
    s.seq_start, s.seq_pos0, s.seq_slot = ints(starts), ints(pos0), slots.int().cuda()
    s.tok_seq = ints([i for i, n in enumerate(news) for _ in range(n)])
    s.tok_pos = ints([p + t for p, n in zip(pos0, news) for t in range(n)])
    s.view = SimpleNamespace(k=s.k, v=s.v, page_table=table.cuda(), page_size=ps, max_pages=max_pages)
    # who shares what: a group's length, the sequence whose page table leads to it, its members' tokens (a sequence that shares
    # nothing is a group of its own, of length 0)
    groups = [[i for i, q in enumerate(seqs) if q[0] == g] for g in range(case["groups"])] + [[i] for i, q in enumerate(seqs) if q[0] < 0]
    toks = [[t for i in of for t in range(starts[i], starts[i + 1])] for of in groups]
    firsts = [0]
    for t in toks:
        firsts.append(firsts[-1] + len(t))
    s.prefix = SimpleNamespace(n_groups=len(groups), most_tokens=max(len(t) for t in toks), most_len=max(seqs[of[0]][1] for of in groups), most_own=max(q[2] + q[3] for q in seqs),
                               group_len=ints([seqs[of[0]][1] for of in groups]), group_seq=ints([of[-1] for of in groups]),
                               tok_first=ints(firsts), toks=ints([t for g in toks for t in g]), seq_skip=ints([q[1] for q in seqs]))
    H, K, D = case["heads"], case["kv_heads"], case["dim"]
    s.q = normal(s.n_tokens, (H + 2 * K) * D)
    s.sinks = torch.randn(H, generator=gen, device="cuda") if case["sink"] else None
    s.sinks_log2 = s.sinks * 1.4426950408889634 if case["sink"] else None
    s.out = torch.empty(s.n_tokens, H * D, dtype=dtype, device="cuda")
    s.scale = D ** -0.5
    # the plain form's lookups: every sequence's table row, and its tokens side by side
    s.rows = table[slots].long().cuda()
    s.place = s.tok_pos.long() - s.seq_pos0.long()[s.tok_seq.long()]
    return s


def run(s):
    if own:
        return _run_own(s)
    return _copy_plain(s) if s.case["op"] in ("fork", "move") else _attend_plain(s)


def _run_own(s):
    from mdma_b200 import ops, ops_tensor
    case = s.case
    if case["op"] in ("fork", "move"):
        ops.copy_pages([s.k, s.v], s.src, s.dst, s.rows if case["op"] == "fork" else None)
        return s.k, s.v
    sizes = (case["heads"], case["kv_heads"], case["dim"], s.scale)
    if case["dtype"] == "bfloat16":
        ops_tensor.prefix_attention(s, s.q, s.view, s.out, *sizes, sink_log2=s.sinks_log2)
    else:
        ops.prefix_attention(s, s.q, s.view, s.out, *sizes, sinks=s.sinks)
    return s.out


def _copy_plain(s):
    """Row r < rows of page dst[i] becomes that of page src[i], at every site."""
    copied = (torch.arange(s.k.shape[2], device="cuda") < s.rows_dev[:, None])[None, :, :, None, None]
    s.k[:, s.dst_dev] = torch.where(copied, s.k[:, s.src_dev], s.k[:, s.dst_dev])
    s.v[:, s.dst_dev] = torch.where(copied, s.v[:, s.src_dev], s.v[:, s.dst_dev])
    return s.k, s.v


def _attend_plain(s):
    """softmax(q k / sqrt(D)) v over the keys up to the query's own, each sequence's keys looked up through its page table; a
    sink is one more exponential in the denominator."""
    case = s.case
    H, K, D, n_seqs = case["heads"], case["kv_heads"], case["dim"], s.n_seqs
    G = H // K
    keys, values = (pool[s.rows].reshape(n_seqs, -1, K, D).permute(0, 2, 1, 3).float() for pool in (s.k, s.v))
    q = torch.zeros(n_seqs, s.max_new, H, D, device="cuda")
    q[s.tok_seq.long(), s.place] = s.q[:, :H * D].reshape(-1, H, D).float()
    q = q.reshape(n_seqs, s.max_new, K, G, D).permute(0, 2, 1, 3, 4).reshape(n_seqs, K, s.max_new * G, D)
    scores = (q @ keys.transpose(2, 3)) * s.scale
    pos = s.seq_pos0[:, None] + torch.arange(s.max_new, device="cuda")
    seen = torch.arange(keys.shape[2], device="cuda") <= pos.repeat_interleave(G, 1)[:, None, :, None]
    scores = scores.masked_fill(~seen, -math.inf)
    sink = s.sinks.reshape(K, 1, G).expand(K, s.max_new, G).reshape(1, K, -1, 1) if case["sink"] else torch.full((1, 1, 1, 1), -math.inf, device="cuda")
    top = torch.maximum(scores.amax(3, keepdim=True), sink)
    weights = torch.exp(scores - top)
    out = (weights @ values) / (weights.sum(3, keepdim=True) + torch.exp(sink - top))
    out = out.reshape(n_seqs, K, s.max_new, G, D).permute(0, 2, 1, 3, 4).reshape(n_seqs, s.max_new, H * D)
    return out[s.tok_seq.long(), s.place].to(s.q.dtype)


# ---- what a pass cannot do without ----------------------------------------------------------------------------------------
def work(case):
    size = 2 if case["dtype"] == "bfloat16" else 4
    if case["op"] in ("fork", "move"):
        src, _, rows = _pairs(case)
        row = case["sites"] * case["kv_heads"] * case["dim"] * 2 * size
        return {"bytes": (sum(dict(zip(src, rows)).values()) + sum(rows)) * row, "flops": 0}
    seqs = _sequences(case)
    H, K, D = case["heads"], case["kv_heads"], case["dim"]
    keys = sum({g: prefix for g, prefix, _, _ in seqs if g >= 0}.values()) + sum(before + new for _, _, before, new in seqs)
    tokens = sum(new for *_, new in seqs)
    seen = sum(new * (prefix + before) + new * (new + 1) // 2 for _, prefix, before, new in seqs)
    return {"bytes": (2 * keys * K * D + 2 * tokens * H * D) * size, "flops": 4 * D * H * seen}


# ---- the definition in 64 bits ---------------------------------------------------------------------------------------------
def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] in ("fork", "move"):
        pools = []
        for pool in (s.k, s.v):
            new = pool.clone()
            for a, b, n in zip(s.src, s.dst, s.rows):
                new[:, b, :n] = pool[:, a, :n]
            pools.append(new)
        return tuple(pools)
    H, K, D, ps = case["heads"], case["kv_heads"], case["dim"], case["page_size"]
    table, starts, before, slots = (t.tolist() for t in (s.view.page_table, s.seq_start, s.seq_pos0, s.seq_slot))
    out = torch.empty(s.n_tokens, H, D, dtype=torch.float64, device="cuda")
    for i in range(s.n_seqs):
        a, b = starts[i], starts[i + 1]
        length = before[i] + b - a
        pages = table[slots[i]][:-(-length // ps)]
        k = torch.cat([s.k[p] for p in pages])[:length].double()
        v = torch.cat([s.v[p] for p in pages])[:length].double()
        later = torch.arange(length, device="cuda")[None, :] > before[i] + torch.arange(b - a, device="cuda")[:, None]
        for h in range(H):
            logit = s.q[a:b, h * D:(h + 1) * D].double() @ k[:, h // (H // K)].T / math.sqrt(D)
            logit[later] = -math.inf
            extra = [s.sinks[h].double().expand(b - a, 1)] if case["sink"] else []
            p = torch.softmax(torch.cat([logit] + extra, 1), 1)[:, :length]
            out[a:b, h] = p @ v[:, h // (H // K)]
    return out.reshape(s.n_tokens, H * D)
