"""Refusals of the verification and page entry points, and their oracles (CPU only: nothing is launched)."""

import ctypes

import numpy as np
import pytest
import torch

from diffspec_mi355x import _ext
from diffspec_mi355x.core.kv_cache import compact_pages, extend_pages, fork_pages, free_pages
from diffspec_mi355x.draft.tree_verification import speculative_accept
from oracle import pages as opages
from oracle import spec as ospec

INVALID, UNSUPPORTED, WORKSPACE = -1, -2, -3


@pytest.fixture()
def dry(dsv_lib):
    dsv_lib.dsv_set_dry_run(1)
    yield dsv_lib
    dsv_lib.dsv_set_dry_run(0)


WS = torch.empty(1 << 22, dtype=torch.uint8)


def ws_ptr():
    return (WS.data_ptr() + 255) // 256 * 256


def spec(lib, T=2, M=4, V=10, nbytes=1 << 21, ws=None, **kw):
    i64 = lambda *s: torch.zeros(s, dtype=torch.int64)  # noqa: E731
    t = dict(target=torch.zeros(T, M, V), draft=i64(T, M), parent=i64(T, M - 1), uniform=torch.zeros(T, M),
             q=torch.zeros(T, M, V), path=i64(T, M), tokens=i64(T, M), info=i64(T, 4))
    t.update(kw)
    d = [_ext.desc(t[k]) for k in ("target", "draft", "parent", "uniform", "q", "path", "tokens", "info")]
    return lib.dsv_spec_accept(*d, ws_ptr() if ws is None else ws, nbytes, None)


def test_spec_accepts_and_refuses(dry):
    assert spec(dry) == 0
    assert spec(dry, q=None) == 0
    assert spec(dry, M=1) == 0
    i64 = lambda *s: torch.zeros(s, dtype=torch.int64)  # noqa: E731
    same = i64(2, 4)
    for bad in [dict(target=torch.zeros(2, 4, 10, dtype=torch.float64).to(torch.int64)), dict(target=torch.zeros(2, 4)),
                dict(target=torch.zeros(2, 10, 4).transpose(1, 2)), dict(draft=torch.zeros(2, 4, dtype=torch.int32)),
                dict(draft=i64(2, 5)), dict(parent=i64(2, 4)), dict(parent=None),
                dict(uniform=torch.zeros(2, 4, dtype=torch.bfloat16)), dict(uniform=torch.zeros(2, 3)),
                dict(q=torch.zeros(2, 4, 10, dtype=torch.bfloat16)), dict(q=torch.zeros(2, 4, 11)), dict(path=i64(2, 3)),
                dict(info=i64(2, 5)), dict(tokens=torch.zeros(2, 4, dtype=torch.int32)), dict(path=same, tokens=same),
                dict(draft=same, path=same), dict(path=i64(1, 4).expand(2, 4))]:
        assert spec(dry, **bad) == INVALID, bad.keys()
    big = torch.zeros(2, 1, 10).expand(2, 1025, 10)
    assert spec(dry, target=big) == UNSUPPORTED
    assert spec(dry, V=50000, ws=0) == WORKSPACE       # (rows shared out over workgroups)
    assert spec(dry, V=50000, nbytes=8) == WORKSPACE
    assert spec(dry, V=50000, ws=ws_ptr() + 16) == WORKSPACE
    assert dry.dsv_spec_workspace_bytes(1, 1025, 10) == 0
    assert dry.dsv_spec_workspace_bytes(1, 4, 1 << 31) == 0
    assert dry.dsv_spec_workspace_bytes((1 << 20) + 1, 4, 10) == 0


def book(B=3, P=8, n_log=4, ps=4, D=8):
    return dict(kv=torch.zeros(1, 2, P, 2, ps, D), table=torch.zeros(B, n_log, dtype=torch.int32),
                ref=torch.zeros(P, dtype=torch.int32), lens=torch.zeros(B, dtype=torch.int32),
                a=torch.zeros(2, dtype=torch.int32), b=torch.zeros(2, dtype=torch.int64),
                new=torch.zeros(B, dtype=torch.int32), info=torch.zeros(3, dtype=torch.int32), ps=ps, nbytes=1 << 21)


def calls(lib, **kw):
    """Return codes of fork, extend, free and compact."""
    t = book()
    t.update(kw)
    d = {k: _ext.desc(v) for k, v in t.items() if isinstance(v, torch.Tensor)}
    return (lib.dsv_pages_fork(d["kv"], d["table"], d["ref"], d["lens"], d["a"], d["b"], d["info"], ws_ptr(), t["nbytes"], None),
            lib.dsv_pages_extend(d["table"], d["ref"], d["lens"], d["new"], t["ps"], d["info"], ws_ptr(), t["nbytes"], None),
            lib.dsv_pages_free(d["table"], d["ref"], d["lens"], d["a"], t["ps"], 0, 0, None),
            lib.dsv_pages_compact(d["kv"], d["table"], d["ref"], d["info"], ws_ptr(), t["nbytes"], None))


def test_pages_accept_and_refuse(dry):
    z = lambda *s, dtype=torch.int32: torch.zeros(s, dtype=dtype)  # noqa: E731
    assert calls(dry) == (0, 0, 0, 0)
    assert calls(dry, a=z(0), b=z(0)) == (0, 0, 0, 0)
    assert calls(dry, lens=z(3, dtype=torch.int64)) == (0, 0, 0, 0)
    everyone = (INVALID,) * 4
    assert calls(dry, table=z(3, 4, dtype=torch.int64)) == everyone
    assert calls(dry, table=z(4, 3).t()) == everyone
    assert calls(dry, table=z(1, 4).expand(3, 4)) == everyone
    assert calls(dry, ref=z(8, dtype=torch.int64)) == everyone
    assert calls(dry, ref=z(16)[::2]) == everyone
    assert calls(dry, lens=z(4))[:3] == everyone[:3]
    assert calls(dry, lens=z(3).float())[:3] == everyone[:3]
    assert calls(dry, info=z(4))[0] == INVALID
    one = z(16)
    assert calls(dry, table=one[:12].view(3, 4), ref=one[8:16]) == everyone
    assert calls(dry, ref=one[:8], info=one[2:5])[3] == INVALID
    assert calls(dry, lens=one[:3], a=one[1:3])[0] == INVALID
    assert calls(dry, b=z(3))[0] == INVALID
    assert calls(dry, new=z(2))[1] == INVALID
    assert calls(dry, ps=6)[1:3] == (UNSUPPORTED, UNSUPPORTED)
    assert calls(dry, nbytes=16)[0] == WORKSPACE
    f = torch.zeros
    assert calls(dry, kv=f(1, 2, 9, 2, 4, 8))[0] == INVALID           # pages differ from refcount's
    assert calls(dry, kv=f(1, 3, 8, 2, 4, 8))[3] == INVALID
    assert calls(dry, kv=f(1, 2, 8, 2, 3, 8))[3] == UNSUPPORTED       # page size
    assert calls(dry, kv=f(1, 2, 8, 2, 4, 6))[3] in (INVALID, UNSUPPORTED)
    assert calls(dry, kv=f(1, 2, 1, 2, 4, 8).expand(1, 2, 8, 2, 4, 8))[3] == INVALID  # pages that share bytes
    assert calls(dry, kv=z(1, 2, 8, 2, 4, 8))[3] == UNSUPPORTED       # dtype
    t = book()
    d = {k: _ext.desc(v) for k, v in t.items() if isinstance(v, torch.Tensor)}
    for window, sinks in [(-1, 0), (4, -1), (0, 3)]:
        assert dry.dsv_pages_free(d["table"], d["ref"], d["lens"], d["a"], 4, window, sinks, None) == INVALID
    assert dry.dsv_pages_workspace_bytes(1 << 31, 1, 1) == 0
    assert dry.dsv_pages_workspace_bytes(8, (1 << 17) + 1, 1) == 0


def test_python_refuses_cpu_tensors(dsv_lib):
    t = book()
    with pytest.raises(RuntimeError):
        fork_pages(t["kv"], t["table"], t["ref"], t["lens"], t["a"], t["b"])
    with pytest.raises(RuntimeError):
        extend_pages(t["table"], t["ref"], t["lens"], t["new"], 4)
    with pytest.raises(RuntimeError):
        free_pages(t["table"], t["ref"], t["lens"], t["a"], 4)
    with pytest.raises(ValueError):
        free_pages(t["table"], t["ref"], t["lens"], t["a"], 4, window=0)
    with pytest.raises(RuntimeError):
        compact_pages(t["kv"], t["table"], t["ref"])
    with pytest.raises(RuntimeError):
        speculative_accept(torch.zeros(1, 2, 4), torch.zeros(1, 2), torch.zeros(1, 1), torch.zeros(1, 2))


def test_integers_beyond_64_bits():
    assert [_ext.i64(x) for x in (0, -5, 2 ** 63 - 1, 2 ** 63, 2 ** 64 + 9, -2 ** 63 - 1, np.int64(7))] == \
        [0, -5, 2 ** 63 - 1, 2 ** 63 - 1, 2 ** 63 - 1, -2 ** 63, 7]


def test_oracle_keeps_the_targets_distribution():
    """The rule itself, over every draft and the numbers integrated: P(first token) is the target's row."""
    rng = np.random.default_rng(0)
    V, grid = 3, 60
    p, q = rng.dirichlet(np.ones(V)), rng.dirichlet(np.ones(V))
    target, dp = np.stack([p] * 3), np.stack([q] * 3)
    mids = (np.arange(grid) + 0.5) / grid
    got = np.zeros(V)
    for x in range(V):
        for y in range(V):
            for u1 in mids:
                for u2 in mids:
                    # The draw integrated exactly: its weights, from the numbers at both ends of each token.
                    path, _ = ospec.speculative_walk(target, [0, x, y], [-1, -1], [0.0, u1, u2], dp)
                    if len(path) > 1:
                        got[[0, x, y][path[1]]] += q[x] * q[y] / grid ** 2
                    else:
                        w1 = np.maximum(p - q, 0)
                        w2 = np.maximum(w1 - w1.sum() * q, 0)
                        got += q[x] * q[y] / grid ** 2 * w2 / w2.sum()
    # Each number is integrated by the midpoint rule: off by half a step of 1/60 for each of the two.
    assert np.abs(got - p).max() < 1.0 / grid


def test_oracle_pages_small():
    kv = np.zeros((1, 2, 6, 1, 2, 8), dtype=np.float32)
    table, ref, lens = [[-1] * 3 for _ in range(3)], [0] * 6, [0] * 3
    assert opages.extend(table, ref, lens, [3, 0, 0], 2) == (2, 0, 0)
    kv[:, :, 1] = 5.0
    assert opages.fork(kv, table, ref, lens, [0], [2], 2) == (1, 0, 0)
    assert table[2] == [0, 2, -1] and ref == [2, 1, 1, 0, 0, 0] and kv[0, 0, 2, 0, 0, 0] == 5.0
    opages.free(table, ref, lens, [0], 2)
    assert ref == [1, 0, 1, 0, 0, 0]
    assert opages.compact(kv, table, ref) == (2, 1, 0)
    assert table[2] == [0, 1, -1] and kv[0, 1, 1, 0, 1, 7] == 5.0
