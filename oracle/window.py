"""Windowed attention with sinks, restated in float64 row by row.

Sums run over the keys that a row sees and over nothing else, so what stands in
other places never enters.
"""

from __future__ import annotations

from typing import List, Optional, Sequence

import numpy as np


def visible(M: int, n: int, window: int, sinks: int, parent: Optional[Sequence[int]] = None) -> List[np.ndarray]:
    """Keys that each of the last M tokens of a sequence of n sees."""
    n0 = n - M
    if parent is None:
        out = []
        for m in range(M):
            p = n0 + m
            keys = np.arange(max(p + 1, 0))
            out.append(keys[(keys > p - window) | (keys < sinks)])
        return out
    if n0 < 0:
        return [np.zeros(0, dtype=np.int64)] * M
    chains = []
    for m in range(M):
        chain, x = [], m
        while 0 <= x < M and len(chain) < M:
            chain.append(x)
            if parent[x] == x:
                break
            x = int(parent[x])
        chains.append(chain)
    out = []
    for m in range(M):
        p = n0 + len(chains[m]) - 1
        pre = np.arange(n0)
        pre = pre[(pre > p - window) | (pre < sinks)]
        own = [n0 + a for h, a in enumerate(chains[m]) if p - h > p - window or p - h < sinks]
        out.append(np.concatenate([pre, np.array(sorted(own), dtype=np.int64)]).astype(np.int64))
    return out


def attend(q: np.ndarray, k: np.ndarray, v: np.ndarray, keys: List[np.ndarray]):
    """One sequence: q [M, H, D], k and v [n, Hk, D], float64.

    Returns out [M, H, D], lse [H, M] and, for error bounds, sum p |v| [M, H, D]
    and the largest sum |q k| / sqrt(D) of a row's keys [H, M].
    """
    M, H, D = q.shape
    G = H // k.shape[1] if k.shape[1] else 1
    out, absum = np.zeros((M, H, D)), np.zeros((M, H, D))
    lse, reach = np.full((H, M), -np.inf), np.zeros((H, M))
    for m in range(M):
        if keys[m].size == 0:
            continue
        kk, vv = np.repeat(k[keys[m]], G, axis=1), np.repeat(v[keys[m]], G, axis=1)  # [n, H, D]
        s = np.einsum("hd,nhd->hn", q[m], kk) / np.sqrt(D)
        reach[:, m] = (np.einsum("hd,nhd->hn", np.abs(q[m]), np.abs(kk)) / np.sqrt(D)).max(1)
        mx = s.max(1, keepdims=True)
        e = np.exp(s - mx)
        z = e.sum(1, keepdims=True)
        out[m] = np.einsum("hn,nhd->hd", e / z, vv)
        absum[m] = np.einsum("hn,nhd->hd", e / z, np.abs(vv))
        lse[:, m] = (mx + np.log(z))[:, 0]
    return out, lse, absum, reach
