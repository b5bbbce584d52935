"""Latent attention: NaN rows and rows of no weight where a sequence's keys are shared out over workgroups, whose
partials are joined.  Bounds: those of test_gpu_latent.py."""

import math

import numpy as np
import pytest
import torch

from diffspec_mi355x import _ext
from diffspec_mi355x.runtime.latent_attention import latent_attn_expanded, latent_attn_with_kvcache
from oracle import latent as oracle
from test_gpu_latent import BF, F16, F32, check, f64, make, make_exp

pytestmark = pytest.mark.gpu


def joins(q, dv, n, tree=False, expanded=False):
    """Partials are written and joined: the call has a workspace."""
    B, M, H, _ = q.shape
    return _ext.load().dsv_latent_workspace_bytes(B, M, H, dv, _ext.desc(q).dtype, n, int(tree), int(expanded)) > 0


# Few rows (a row a workgroup of the join), some, many; more sequences than ranges; a tree.
@pytest.mark.parametrize("dtype", [BF, F16, F32])
@pytest.mark.parametrize("B,M,H,n,tree", [(1, 1, 16, 3001, False), (2, 2, 5, 5000, False), (40, 1, 16, 700, False),
                                          (40, 1, 256, 700, False), (100, 1, 256, 300, False), (3, 9, 4, 2000, True)])
def test_absorbed_nan_query(gpu, dtype, B, M, H, n, tree):
    """Of one sequence, a head's query is NaN: its row comes out NaN, every other row as without it."""
    lens = [n - 3 * b for b in range(B)]
    q, kv, table, sl, parent, rows = make(dtype, B, M, H, 256, 32, 16, lens, tree, seed=B + H)
    assert joins(q, 256, table.shape[1] * 16, tree)
    b, m, h = B // 2, M // 2, H // 3
    q[b, m, h, 7] = math.nan
    out, lse = latent_attn_with_kvcache(q, kv, 256, 0.06, cache_seqlens=sl, page_table=table, parent=parent,
                                        return_softmax_lse=True)
    assert torch.isnan(out[b, m, h].float()).all() and torch.isnan(lse[b, h, m])
    bad = torch.isnan(out.float()).any(-1)
    assert int(bad.sum()) == 1 and int(torch.isnan(lse).sum()) == 1
    for y in sorted({0, b, B - 1}):
        x = f64(rows[y])
        seen = oracle.visible(M, lens[y], parent[y].tolist() if tree else None)
        for z in sorted({0, h, H - 1}):
            keep = [i for i in range(M) if (y, i, z) != (b, m, h)]
            if keep:
                ref = oracle.attention(f64(q[y, keep, z]), x, x[:, :256], 0.06, [seen[i] for i in keep])
                check(out[:, keep], lse[:, :, keep], y, z, ref, 288, dtype, lens[y], np.abs(x).max())


@pytest.mark.parametrize("dtype", [BF, F16, F32])
@pytest.mark.parametrize("M,tree", [(1, False), (4, False), (4, True)])
@pytest.mark.parametrize("kind", ["nan", "no weight"])
def test_absorbed_last_key_alone(gpu, dtype, M, tree, kind):
    """Every tile a range of its own, the last one with one key, which one row sees: a NaN key spoils that row, an infinite
    entry of a score of -inf its own column (0 * inf), and other rows not at all."""
    n, H, dc, D = 64 * 10 + 1, 16, 256, 288
    q, kv1, _, sl, _, rows = make(dtype, 1, M, H, dc, 32, 0, [n], False, seed=M)
    kv = torch.full((1, 8192, D), math.nan, dtype=dtype, device=gpu)  # (128 tiles: ranges for them, of which 11 are used)
    kv[:, :n] = kv1
    parent = torch.tensor([-1] + [0] * (M - 1), device=gpu) if tree else None
    assert joins(q, dc, 8192, tree)
    q[..., 9] = -q[..., 9].abs() - 0.25
    kv[0, n - 1, 9] = math.nan if kind == "nan" else math.inf
    out, lse = latent_attn_with_kvcache(q, kv, dc, 0.05, cache_seqlens=sl, parent=parent, return_softmax_lse=True)
    x = f64(kv[0, :n])
    x[n - 1] = 0
    seen = oracle.visible(M, n, parent.tolist() if tree else None)
    clean = [m for m in range(M - 1)]
    assert all(n - 1 not in seen[m] for m in clean)
    for h in range(H):
        if clean:
            ref = oracle.attention(f64(q[0, clean, h]), x, x[:, :dc], 0.05, [seen[m] for m in clean])
            check(out[:, clean], lse[:, :, clean], 0, h, ref, D, dtype, n, np.abs(x).max())
        if kind == "nan":
            assert torch.isnan(out[0, M - 1, h].float()).all() and torch.isnan(lse[0, h, M - 1])
        else:
            assert torch.isnan(out[0, M - 1, h, 9].float())
            keep = [c for c in range(dc) if c != 9]
            ref = oracle.attention(f64(q[0, M - 1:, h]), x, x[:, :dc], 0.05, [seen[M - 1][:-1]])
            ref = {**ref, "out": ref["out"][:, keep], "mass": ref["mass"][:, keep]}
            check(out[:, M - 1:][..., keep], lse[:, :, M - 1:], 0, h, ref, D, dtype, n, np.abs(x).max())


@pytest.mark.parametrize("dtype", [BF, F16, F32])
@pytest.mark.parametrize("M,causal", [(1, True), (5, True), (5, False)])
@pytest.mark.parametrize("kind", ["query", "nan", "no weight"])
def test_expanded(gpu, dtype, M, causal, kind):
    """The same with keys and values per head: a NaN query, a NaN last key, and one of no weight with an infinite value."""
    n, N, H, dn, dr = 641, 8192, 2, 64, 32
    q, k, pe, v, sl = make_exp(dtype, 1, M, N, H, dn, dr, [n], seed=M)
    assert joins(q, dn, N, expanded=True)
    q[..., 3] = -q[..., 3].abs() - 0.25
    hit = [M - 1] if causal else list(range(M))  # (rows that see the last key)
    if kind == "query":
        hit = [M - 1]
        q[0, M - 1, 0, 5] = math.nan
    elif kind == "nan":
        k[0, n - 1, 0, 3] = math.nan
    else:
        k[0, n - 1, 0, 3] = math.inf
        v[0, n - 1, 0, 7] = math.inf
    out, lse = latent_attn_expanded(q, k, pe, v, cache_seqlens=sl, causal=causal, return_softmax_lse=True)
    seen = oracle.visible(M, n, causal=causal)
    scale = (dn + dr) ** -0.5
    for h in range(H):
        x, y = np.concatenate([f64(k[0, :n, h]), f64(pe[0, :n])], -1), f64(v[0, :n, h])
        rest = [m for m in range(M) if h == 1 or m not in hit]
        if h == 0 and kind != "query":
            x[n - 1], y[n - 1] = 0, 0  # (seen by none of the rest)
        if rest:
            ref = oracle.attention(f64(q[0, rest, h]), x, y, scale, [seen[m] for m in rest])
            check(out[:, rest], lse[:, :, rest], 0, h, ref, dn + dr, dtype, n, np.abs(y).max())
    got = out[0, hit, 0].float()
    if kind != "no weight":
        assert torch.isnan(got).all() and torch.isnan(lse[0, 0, hit]).all()
        return
    assert torch.isnan(got[:, 7]).all()
    keep = [c for c in range(dn) if c != 7]
    ref = oracle.attention(f64(q[0, hit, 0]), np.concatenate([f64(k[0, :n, 0]), f64(pe[0, :n])], -1)[:-1], f64(v[0, :n - 1, 0]),
                           scale, [seen[m][seen[m] < n - 1] for m in hit])
    ref = {**ref, "out": ref["out"][:, keep], "mass": ref["mass"][:, keep]}
    check(out[:, hit][..., keep], lse[:, :, hit], 0, 0, ref, dn + dr, dtype, n, np.abs(f64(v[0, :n - 1, 0])).max())
