"""Page bookkeeping of a paged KV cache on Python lists: fork, extend, free, compact.

Each function changes its arguments as the device operators change theirs and
returns the same three numbers.  ``kv`` is a numpy pool [L, 2, P, Hk, page, D].
"""

from __future__ import annotations

from typing import List, Optional, Sequence, Tuple

import numpy as np


def fork(kv: np.ndarray, table: List[List[int]], ref: List[int], lens: List[int], parents: Sequence[int],
         children: Sequence[int], ps: int) -> Tuple[int, int, int]:
    B, P, n_log = len(table), len(ref), len(table[0])
    bad, seen = 0, set()
    roots = set()
    for a, c in zip(parents, children):
        ok = 0 <= a < B and 0 <= c < B and a != c
        if ok:
            ok = 0 <= lens[a] <= n_log * ps and lens[c] == 0 and c not in seen
            seen.add(c)
            roots.add(a)
        bad += not ok
    bad += sum(1 for c in children if 0 <= c < B and c in roots)
    if bad:
        return 0, 0, bad
    copies = []
    for i, a in enumerate(parents):
        if lens[a] % ps and 0 <= table[a][lens[a] // ps] < P:
            copies.append(i)
    free = [p for p in range(P) if ref[p] == 0]
    if len(free) < len(copies):
        return 0, len(copies) - len(free), 0
    own = dict(zip(copies, free))
    for i, (a, c) in enumerate(zip(parents, children)):
        n = lens[a]
        for j in range(n_log):
            page = table[a][j] if j * ps < n else -1
            if (j + 1) * ps <= n:
                if 0 <= page < P:
                    ref[page] += 1
            elif j * ps < n and i in own:
                kv[:, :, own[i]] = kv[:, :, page]
                page = own[i]
                ref[page] = 1
            table[c][j] = page
        lens[c] = n
    return len(copies), 0, 0


def extend(table: List[List[int]], ref: List[int], lens: List[int], new: Sequence[int], ps: int) -> Tuple[int, int, int]:
    n_log = len(table[0])
    grow = [b for b in range(len(table)) if new[b] > lens[b]]
    bad = sum(1 for b in grow if lens[b] < 0 or new[b] > n_log * ps)
    if bad:
        return 0, 0, bad
    slots = [(b, j) for b in grow for j in range(-(-lens[b] // ps), -(-new[b] // ps)) if not 0 <= table[b][j] < len(ref)]
    free = [p for p in range(len(ref)) if ref[p] == 0]
    if len(free) < len(slots):
        return 0, len(slots) - len(free), 0
    for (b, j), p in zip(slots, free):
        table[b][j] = p
        ref[p] = 1
    for b in grow:
        lens[b] = new[b]
    return len(slots), 0, 0


def free(table: List[List[int]], ref: List[int], lens: List[int], seqs: Sequence[int], ps: int,
         window: Optional[int] = None, sinks: int = 0) -> None:
    for s in seqs:
        if not 0 <= s < len(table):
            continue
        for j, page in enumerate(table[s]):
            if window is not None:
                # A token n is out of sight of the next one (position len) when n <= len - window and n >= sinks.
                if not all(n >= sinks and n <= lens[s] - window for n in range(j * ps, (j + 1) * ps)):
                    continue
            if 0 <= page < len(ref):
                ref[page] = max(ref[page] - 1, 0) if ref[page] > 0 else ref[page]
            table[s][j] = -1
        if window is None:
            lens[s] = 0


def compact(kv: np.ndarray, table: List[List[int]], ref: List[int]) -> Tuple[int, int, int]:
    used = [p for p in range(len(ref)) if ref[p] > 0]
    holes = [p for p in range(len(used)) if ref[p] <= 0]
    to = dict(zip([p for p in used if p >= len(used)], holes))
    for s, d in to.items():
        kv[:, :, d] = kv[:, :, s]
        ref[d], ref[s] = ref[s], 0
    for row in table:
        row[:] = [to.get(p, p) for p in row]
    return len(used), len(to), 0
