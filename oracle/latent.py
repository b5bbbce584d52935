"""Serving over a cache of one latent vector per token, restated in float64.

Attention sums run over the keys that a row sees and over nothing else, so what
stands in other places never enters.
"""

from __future__ import annotations

from typing import Dict, List, Optional, Sequence

import numpy as np


def visible(M: int, n: int, parent: Optional[Sequence[int]] = None, causal: bool = True) -> List[np.ndarray]:
    """Keys that each of the last M tokens of a sequence of n sees."""
    n0 = n - M
    if not causal:
        return [np.arange(n)] * M
    if parent is None:
        return [np.arange(max(n0 + m + 1, 0)) for m in range(M)]
    if n0 < 0:
        return [np.zeros(0, dtype=np.int64)] * M
    out = []
    for m in range(M):
        chain, x = [], m
        while 0 <= x < M and len(chain) < M:
            chain.append(x)
            p = int(parent[x])
            x = -1 if p == x else p
        out.append(np.concatenate([np.arange(n0), n0 + np.array(sorted(set(chain)), dtype=np.int64)]))
    return out


def attention(q: np.ndarray, keys: np.ndarray, values: np.ndarray, scale: float, seen: List[np.ndarray]) -> Dict[str, np.ndarray]:
    """One head: q [M, D], keys [n, D], values [n, Dv]; seen[m] lists row m's keys.

    Beside out [M, Dv] and lse [M] come the weighted means of |v| ("mass" [M, Dv]) and the
    largest scale * sum |q_i k_i| of a seen key ("reach" [M]), by which errors are bounded.
    """
    M = q.shape[0]
    out, mass = np.zeros((M, values.shape[1])), np.zeros((M, values.shape[1]))
    lse, reach = np.full(M, -np.inf), np.zeros(M)
    with np.errstate(invalid="ignore", over="ignore"):
        for m in range(M):
            if len(seen[m]) == 0:
                continue
            k, v = keys[seen[m]], values[seen[m]]
            s = (k @ q[m]) * scale
            reach[m] = (np.abs(k) @ np.abs(q[m])).max() * scale
            top = s.max()
            e = np.exp(s - top)
            z = e.sum()
            out[m], mass[m], lse[m] = (e @ v) / z, (e @ np.abs(v)) / z, top + np.log(z)
    return {"out": out, "lse": lse, "mass": mass, "reach": reach}


def token_slots(table, lens, news, page: int, cap: int, seqs=None):
    """The lists of token_slots on Python integers."""
    B, n_log = len(table), len(table[0]) if len(table) else 0
    seqs = list(range(len(news))) if seqs is None else list(seqs)
    slots, pos, req, cu, block, out = [-1] * cap, [-1] * cap, [-1] * cap, [0], [], []
    for i, (s, k) in enumerate(zip(seqs, news)):
        n = min(max(int(lens[s]), 0), n_log * page) if 0 <= s < B else 0
        k = min(max(int(k), 0), n)
        for t in range(cu[-1], min(cu[-1] + k, cap)):
            p = n - k + t - cu[-1]
            pg = int(table[s][p // page])
            slots[t], pos[t], req[t] = (pg * page + p % page if pg >= 0 else -1), p, i
        cu.append(cu[-1] + k)
        used = -(-n // page)
        block.append([int(table[s][j]) if j < used else -1 for j in range(n_log)])
        out.append(n)
    return slots, pos, req, [min(x, 2 ** 31 - 1) for x in cu], block, out


def rotate(x: np.ndarray, cos: np.ndarray, sin: np.ndarray, interleaved: bool) -> np.ndarray:
    p = np.empty_like(x)
    if interleaved:
        p[..., 0::2], p[..., 1::2] = -x[..., 1::2], x[..., 0::2]
    else:
        h = x.shape[-1] // 2
        p[..., :h], p[..., h:] = -x[..., h:], x[..., :h]
    return x * cos + p * sin


def latent_rows(c: np.ndarray, pe: np.ndarray, weight: Optional[np.ndarray], eps: float, cos, sin, interleaved: bool) -> np.ndarray:
    if weight is not None:
        c = c / np.sqrt((c * c).mean(-1, keepdims=True) + eps) * weight
    if cos is not None:
        pe = rotate(pe, cos, sin, interleaved)
    return np.concatenate([c, pe], -1)
