"""Verification of drafted tokens from given random numbers, restated for one tree in float64.

Written from the rule itself: sequential rejection with an explicit residual
distribution per rejected sibling (the kernels carry one scalar instead).
"""

from __future__ import annotations

from typing import List, Optional, Sequence, Tuple

import numpy as np


def clean(row: np.ndarray) -> np.ndarray:
    """Probability entries as the operator reads them: negative, infinite and NaN ones are 0."""
    r = np.asarray(row, dtype=np.float64)
    return np.where(np.isfinite(r) & (r > 0), r, 0.0)


def unit(u: float) -> float:
    """A given number clamped into [0, 1) (the largest fp32 below 1)."""
    u = float(u)
    if not u >= 0.0:
        return 0.0
    return min(u, float(np.nextafter(np.float32(1.0), np.float32(0.0))))


def draw(w: np.ndarray, u: float) -> int:
    """First index whose cumulative weight exceeds u times the total."""
    cdf = np.cumsum(w)
    i = int(np.searchsorted(cdf, unit(u) * cdf[-1], side="right"))
    return min(i, int(np.flatnonzero(w)[-1]))


def speculative_walk(target: np.ndarray, draft: Sequence[int], parent_ref: Sequence[int], uniform: Sequence[float],
                     draft_probs: Optional[np.ndarray] = None) -> Tuple[List[int], int]:
    """(path node ids root first, next token)."""
    M, V = target.shape
    kids: List[List[int]] = [[] for _ in range(M)]
    for k, r in enumerate(parent_ref):
        r = int(r)
        if r == -1 or r == k:
            kids[0].append(k + 1)
        elif 0 <= r < M - 1:
            kids[r + 1].append(k + 1)
    node, path = 0, [0]
    while True:
        p = clean(target[node])
        q = clean(draft_probs[node]) if draft_probs is not None else None
        w, mass, hit = p.copy(), 1.0, None
        for k in kids[node]:
            x = int(draft[k])
            inside = 0 <= x < V
            wx = w[x] if inside else 0.0
            qx = (q[x] if inside else 0.0) if q is not None else 1.0
            if unit(uniform[k]) * mass * qx < wx:
                hit = k
                break
            if q is not None:
                w = np.maximum(w - mass * q, 0.0)
                mass = float(np.sum(w))
            elif inside:
                mass -= wx
                w[x] = 0.0
        if hit is None:
            break
        node = hit
        path.append(node)
    if not w.sum() > 0:
        w = p
    return path, (draw(w, uniform[0]) if w.sum() > 0 else 0)
