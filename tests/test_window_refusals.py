"""Refusals and key geometry of the windowed attention (CPU only: nothing is launched)."""

import time

import numpy as np
import pytest
import torch

from diffspec_mi355x import _ext
from diffspec_mi355x.runtime.window_attention import window_attn_with_kvcache
from oracle import window as oracle

INVALID, UNSUPPORTED, WORKSPACE = -1, -2, -3
WS = torch.empty(1 << 24, dtype=torch.uint8)


@pytest.fixture()
def dry(dsv_lib):
    dsv_lib.dsv_set_dry_run(1)
    yield dsv_lib
    dsv_lib.dsv_set_dry_run(0)


def call(lib, B=2, M=3, H=4, Hk=2, D=64, N=40, window=9, sinks=2, n_keys=-1, nbytes=1 << 23, ws=None, **kw):
    sizes = dict(q=(B, M, H, D), k=(B, N, Hk, D), v=(B, N, Hk, D), out=(B, M, H, D), lse=(B, H, M))
    t = {x: kw[x] if x in kw else torch.zeros(sizes[x]) if x in sizes else None
         for x in ("q", "k", "v", "table", "lens", "parent", "out", "lse")}
    d = {x: _ext.desc(y) for x, y in t.items()}
    ptr = (WS.data_ptr() + 255) // 256 * 256 if ws is None else ws
    return lib.dsv_window_attention(d["q"], d["k"], d["v"], d["table"], d["lens"], n_keys, window, sinks, d["parent"],
                                    d["out"], d["lse"], ptr, nbytes, None)


def test_accepts_and_refuses(dry):
    f, i32 = torch.zeros, lambda *s: torch.zeros(s, dtype=torch.int32)
    paged = dict(k=f(7, 2, 8, 64), v=f(7, 2, 8, 64), table=i32(2, 5))
    assert call(dry) == 0
    assert call(dry, lse=None) == 0
    assert call(dry, n_keys=10 ** 12, window=1 << 62, sinks=1 << 62) == 0
    assert call(dry, **paged) == 0
    assert call(dry, **{**paged, "table": torch.zeros(5, dtype=torch.int64)}) == 0
    assert call(dry, parent=i32(3), lens=i32(2)) == 0
    assert call(dry, parent=i32(2, 3).long(), lens=i32(2).long()) == 0
    assert call(dry, out=torch.zeros(2, 3, 4, 64, dtype=torch.bfloat16)) == 0
    for bad in [dict(window=0), dict(window=-4), dict(sinks=-1), dict(Hk=3), dict(k=f(2, 40, 2, 128)), dict(v=f(2, 41, 2, 64)),
                dict(k=f(2, 40, 2, 64).bfloat16()), dict(q=f(2, 3, 64)), dict(out=f(2, 3, 4, 32)), dict(lse=f(2, 3, 4)),
                dict(lse=f(2, 4, 3).double().to(torch.int64)), dict(lens=i32(3)), dict(lens=f(2)), dict(lens=i32(4)[::2]),
                dict(parent=i32(4)), dict(parent=i32(3, 3)), dict(parent=f(3)), dict(table=i32(2, 5)),
                {**paged, "table": i32(3, 5)}, {**paged, "table": f(2, 5)}, {**paged, "table": i32(5, 2).t()},
                dict(q=f(2, 3, 4, 65)[..., 1:]), dict(q=f(2 * 3 * 4 * 64 + 1)[1:].view(2, 3, 4, 64)),
                {**paged, "k": f(6, 2, 8, 64)}]:
        assert call(dry, **bad) == INVALID, bad.keys()
    assert call(dry, D=96) == UNSUPPORTED
    assert call(dry, **{**paged, "k": f(7, 2, 6, 64), "v": f(7, 2, 6, 64)}) == UNSUPPORTED
    big = torch.zeros(1, 1, 1, 64)
    assert call(dry, B=1, M=1025, parent=i32(1025)) == UNSUPPORTED
    assert call(dry, B=1, M=(1 << 24) + 1, H=1, Hk=1, q=big.expand(1, (1 << 24) + 1, 1, 64),
                out=big.clone().expand(1, (1 << 24) + 1, 1, 64), lse=None) == UNSUPPORTED
    wide, kv = big.expand(1 << 20, 1, 8, 64), big.expand(1 << 20, 40, 8, 64)  # 2^23 workgroups
    assert call(dry, B=1 << 20, M=1, H=8, Hk=8, q=wide, out=big.clone().expand(1 << 20, 1, 8, 64),
                k=kv, v=kv, lse=None) == UNSUPPORTED
    many = dict(B=1, N=8192, window=8192)  # (keys shared out over workgroups)
    assert call(dry, **many) == 0
    assert call(dry, ws=0, **many) == WORKSPACE
    assert call(dry, nbytes=0, **many) == WORKSPACE
    assert call(dry, ws=(WS.data_ptr() + 255) // 256 * 256 + 64, **many) == WORKSPACE
    assert call(dry, ws=0, nbytes=0) == 0  # none needed
    q = f(2, 3, 4, 64)
    assert call(dry, q=q, out=q) == INVALID
    assert call(dry, lse=q.view(-1)[:24].view(2, 4, 3), q=q) == INVALID


@pytest.mark.parametrize("seed", range(40))
def test_every_address_and_key(dry, seed):
    """The kernels' key geometry and addresses, walked on the host: in range, every seen key in one tile."""
    rng = np.random.default_rng(seed)
    pick = lambda *x: x[int(rng.integers(len(x)))]  # noqa: E731
    B, Hk, G, D = pick(1, 3), pick(1, 2), pick(1, 2, 7, 16), pick(64, 128)
    M, N = int(pick(1, 2, 5, 31, 64, 200)), int(pick(1, 33, 200, 700))
    dt = pick(torch.bfloat16, torch.float16, torch.float32)
    kw = dict(B=B, M=M, H=Hk * G, Hk=Hk, D=D, window=int(pick(1, 7, 32, 100, 1000)), sinks=int(pick(0, 1, 31, 33, 90)),
              q=torch.zeros(B, M, Hk * G, D, dtype=dt), nbytes=(1 << 24) - 256)
    if rng.random() < 0.5:
        page = int(pick(1, 4, 16, 64))
        n_log = -(-N // page)
        kv = torch.zeros(2, 5, Hk, page, D, dtype=dt)
        kw.update(k=kv[0], v=kv[1], table=torch.zeros((B, n_log) if rng.random() < 0.7 else (n_log,), dtype=pick(torch.int32, torch.int64)))
    else:
        kv = torch.zeros(2, B, N, Hk, D + 8, dtype=dt)[..., :D]
        kw.update(k=kv[0], v=kv[1])
    if rng.random() < 0.8:
        kw.update(lens=torch.zeros(B, dtype=torch.int32))
    if rng.random() < 0.4:
        kw.update(parent=torch.zeros((B, M), dtype=torch.int64))
    if rng.random() < 0.3:
        kw.update(n_keys=max(1, N // 2))
    assert call(dry, **kw) == 0, _ext.last_error()
    assert dry.dsv_dry_run_checks() > 0


@pytest.mark.parametrize("M", [1, 64])
def test_dry_run_of_the_longest_cache(dry, M):
    """2^30 keys: the tiles' addresses are walked, not every key of the cache."""
    kv, q = torch.zeros(1, 1, 1, 64).expand(1, 1 << 30, 2, 64), torch.zeros(1, M, 4, 64)
    t0 = time.monotonic()
    assert call(dry, B=1, M=M, q=q, k=kv, v=kv, lens=torch.zeros(1, dtype=torch.int32), window=512, sinks=4) == 0, _ext.last_error()
    assert dry.dsv_dry_run_checks() > 0
    assert time.monotonic() - t0 < 20.0  # (milliseconds; minutes if every key were walked)


def test_workspace_sizes(dsv_lib):
    n = dsv_lib.dsv_window_workspace_bytes
    assert n(1, 1, 32, 8, 128, _ext.DSV_BF16, 50000, 8192, 4, 0) > 0
    assert n(1, 1, 32, 8, 128, _ext.DSV_BF16, 50000, 512, 4, 0) == 0
    for bad in [(0, 1, 4, 2, 64, 0, 10, 4, 0, 0), (1, 0, 4, 2, 64, 0, 10, 4, 0, 0), (1, 1, 4, 3, 64, 0, 10, 4, 0, 0),
                (1, 1, 4, 2, 80, 0, 10, 4, 0, 0), (1, 1, 4, 2, 64, 3, 10, 4, 0, 0), (1, 1, 4, 2, 64, 0, -1, 4, 0, 0),
                (1, 1, 4, 2, 64, 0, 10, 0, 0, 0), (1, 1, 4, 2, 64, 0, 10, 4, -1, 0), (1, 1025, 4, 2, 64, 0, 10, 4, 0, 1),
                ((1 << 20) + 1, 1, 4, 2, 64, 0, 10, 4, 0, 0), (1 << 20, 1, 8, 8, 64, 0, 10, 4, 0, 0)]:
        assert n(*bad) == 0, bad


@pytest.mark.parametrize("big", [1 << 30, 1 << 62, (1 << 63) - 70, (1 << 63) - 2, (1 << 63) - 1])
@pytest.mark.parametrize("M,tree", [(1, False), (5, False), (64, True), (300, False)])
def test_workspace_of_a_window_beyond_every_key(dry, M, tree, big):
    """The queried number of bytes is what the call asks for, up to the largest window and sinks; all mean every key."""
    N = 50000
    kv, q = torch.zeros(1, 1, 1, 128, dtype=torch.bfloat16).expand(1, N, 8, 128), torch.zeros(1, M, 32, 128, dtype=torch.bfloat16)
    size = lambda w, s: dry.dsv_window_workspace_bytes(1, M, 32, 8, 128, _ext.DSV_BF16, N, w, s, int(tree))  # noqa: E731
    assert size(big, 0) == size(N + M, 0) > 0
    for window, sinks in [(big, 0), (9, big), (big, big)]:
        n = size(window, sinks)
        ws = torch.empty(n + 256, dtype=torch.uint8)
        ptr = (ws.data_ptr() + 255) // 256 * 256
        assert call(dry, B=1, M=M, H=32, Hk=8, D=128, q=q, k=kv, v=kv, window=window, sinks=sinks, nbytes=n, ws=ptr, lse=None,
                    out=torch.zeros_like(q), parent=torch.zeros(M, dtype=torch.int32) if tree else None) == 0, _ext.last_error()


def test_python_refusals(dsv_lib):
    q, k = torch.zeros(1, 2, 4, 64), torch.zeros(1, 9, 2, 64)
    with pytest.raises(RuntimeError):
        window_attn_with_kvcache(q, k, k, 4)


def test_oracle_against_a_dense_mask():
    """The oracle's visible keys against the definition as one mask."""
    rng = np.random.default_rng(0)
    for _ in range(200):
        M, n = int(rng.integers(1, 9)), int(rng.integers(0, 30))
        W, S = int(rng.integers(1, 12)), int(rng.integers(0, 8))
        got = oracle.visible(M, n, W, S)
        for m in range(M):
            p = n - M + m
            assert got[m].tolist() == [j for j in range(n) if j <= p and (j > p - W or j < S)]
        par = [-1] + [int(rng.integers(-1, i)) for i in range(1, M)]
        got = oracle.visible(M, n, W, S, par)
        depth = [0] * M
        for i in range(1, M):
            depth[i] = 0 if par[i] < 0 else depth[par[i]] + 1
        anc = np.eye(M, dtype=bool)
        for i in range(1, M):
            if par[i] >= 0:
                anc[i] |= anc[par[i]]
        n0 = n - M
        for m in range(M):
            want = []
            for j in range(n) if n0 >= 0 else []:
                pos = j if j < n0 else n0 + depth[j - n0]
                if (j < n0 or anc[m, j - n0]) and (pos > n0 + depth[m] - W or pos < S):
                    want.append(j)
            assert got[m].tolist() == want
