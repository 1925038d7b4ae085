"""Which sequences of a step begin with the same tokens, as the attention kernels for shared prefixes take it.

Every sequence of a step belongs to one group; the members' first `length` tokens lie in pages that their page tables share
(the rows of a partly filled last page may be copies, one a member).  A sequence that shares nothing is a group of
its own, of length 0.  Device tables (int32): `group_len` and `group_seq` [groups], a member whose page table leads to the prefix;
`tok_first` [groups + 1] and `toks` [tokens], the members' token rows, group after group; `seq_skip` [sequences], the
length of each sequence's prefix.  The host keeps the upper bounds that kernels size their grids by.
"""
from __future__ import annotations

from typing import Optional, Sequence

import numpy as np
import torch


class PrefixGroups:
    FIELDS = ("group_len", "group_seq", "tok_first", "toks", "seq_skip")

    def __init__(self, shared: Sequence[tuple[int, Sequence[int]]], pos0: Sequence[int], new: Sequence[int],
                 device: Optional[torch.device] = None):
        """`shared`: (length, numbers of the sequences that share it); `pos0`, `new`: positions that every sequence of the step
        holds already and the tokens it brings.  With a `device` the tables are uploaded; else see `words` and `bind`."""
        n = len(pos0)
        if len(new) != n:
            raise ValueError(f"{n} sequences, {len(new)} token counts")
        skip = [0] * n
        taken: set[int] = set()
        groups: list[tuple[int, list[int]]] = []
        for length, members in shared:
            members = [int(m) for m in members]
            if not members or length < 0:
                raise ValueError(f"a prefix of {length} tokens shared by {len(members)} sequences")
            for m in members:
                if not 0 <= m < n or m in taken:
                    raise ValueError(f"sequence {m} is not of this step, or shares two prefixes")
                if length > pos0[m]:
                    raise ValueError(f"sequence {m} holds {pos0[m]} tokens, its shared prefix is {length} long")
                taken.add(m)
                skip[m] = int(length)
            groups.append((int(length), members))
        groups += [(0, [m]) for m in range(n) if m not in taken]
        starts = np.concatenate([[0], np.cumsum(np.asarray(new, dtype=np.int64))])
        toks = [np.arange(starts[m], starts[m + 1]) for _, members in groups for m in members]
        sizes = [int(sum(starts[m + 1] - starts[m] for m in members)) for _, members in groups]
        self.n_groups = len(groups)
        # what plans go by: groups with a prefix, the members of the largest, the keys that all members see of their prefixes (an
        # engine counts those that have ended, too)
        self.n_shared = sum(1 for length, _ in groups if length)
        self.most_members = max((len(members) for length, members in groups if length), default=0)
        self.shared_keys = sum(length * len(members) for length, members in groups)
        self.most_tokens = max(sizes, default=0)
        self.most_len = max((length for length, _ in groups), default=0)
        self.skips = skip
        self.most_own = max((p + t - s for p, t, s in zip(pos0, new, skip)), default=0)
        self._host = {"group_len": [length for length, _ in groups], "group_seq": [members[0] for _, members in groups],
                      "tok_first": np.concatenate([[0], np.cumsum(sizes)]) if groups else [0],
                      "toks": np.concatenate(toks) if toks else [], "seq_skip": skip}
        if device is not None:
            self.bind(torch.from_numpy(self.words()).to(device))

    def words(self) -> np.ndarray:
        """The tables one behind the other, for an upload in one piece."""
        return np.concatenate([np.asarray(self._host[f], dtype=np.int32) for f in self.FIELDS])

    def bind(self, words: torch.Tensor) -> None:
        """`words`: where the device holds `words()`."""
        at = 0
        for f in self.FIELDS:
            n = len(self._host[f])
            setattr(self, f, words[at:at + n])
            at += n
