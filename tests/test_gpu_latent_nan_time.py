"""Latent attention: which NaN and infinite values cost a second pass over a block's rows, and what comes out."""

import math

import numpy as np
import pytest
import torch

from diffspec_mi355x.runtime.latent_attention import latent_attn_expanded, latent_attn_with_kvcache
from oracle import latent as oracle
from test_gpu_latent import BF, F16, F32, check, f64, make, make_exp

pytestmark = pytest.mark.gpu


def micros(call):
    call()
    best = math.inf
    for _ in range(5):
        a, b = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
        a.record()
        call()
        b.record()
        torch.cuda.synchronize()
        best = min(best, a.elapsed_time(b))
    return best * 1e3


@pytest.mark.parametrize("dtype,B,M,H,dc,dr", [(BF, 32, 1, 128, 512, 64), (BF, 1, 128, 128, 512, 64), (F16, 4, 64, 16, 256, 32),
                                               (F32, 1, 64, 16, 512, 64)])
@pytest.mark.parametrize("tree", [False, True])
@pytest.mark.parametrize("kind", ["queries", "token of the prefix"])
def test_nan_that_needs_no_second_pass(gpu, dtype, B, M, H, dc, dr, tree, kind):
    """NaN queries, and a NaN token that all rows see, take about as long as sound ones (a second pass took 15 to 270
    times as long), and everything that they reach is NaN."""
    n = 1000
    q, kv, _, sl, parent, _ = make(dtype, B, M, H, dc, dr, 0, [n - 3] * B, tree, seed=1)
    kv = torch.cat([kv, torch.zeros((B, 3, dc + dr), dtype=dtype, device=gpu)], 1)
    sound = micros(lambda: latent_attn_with_kvcache(q, kv, dc, 0.04, cache_seqlens=sl, parent=parent))
    if kind == "queries":
        q = q * math.nan
    else:
        kv[:, n - 3 - M - (0 if M > 1 else -1) - 1] = math.nan
    call = lambda: latent_attn_with_kvcache(q, kv, dc, 0.04, cache_seqlens=sl, parent=parent, return_softmax_lse=True)  # noqa: E731
    took = micros(call)
    out, lse = call()
    assert torch.isnan(out.float()).all() and torch.isnan(lse).all()
    assert took <= 5 * sound + 50, (sound, took)


@pytest.mark.parametrize("dtype", [BF, F16, F32])
@pytest.mark.parametrize("H", [1, 5, 40])
@pytest.mark.parametrize("n", [70, 64, 130, 5000])
def test_nan_query_beside_an_infinite_hidden_value(gpu, dtype, H, n):
    """One row's query is NaN and the last token infinite: the NaN row, the rows that see the token, and those that do not."""
    M, dc = 6, 256
    q, kv, _, sl, _, rows = make(dtype, 1, M, H, dc, 32, 0, [n], False, seed=H)
    q[0, 1, 0, 5] = math.nan
    q[..., 4] = q[..., 4].abs() + 0.5
    kv[0, n - 1, 4] = -math.inf  # (no weight: its column alone)
    out, lse = latent_attn_with_kvcache(q, kv, dc, 0.05, cache_seqlens=sl, return_softmax_lse=True)
    assert torch.isnan(out[0, 1, 0].float()).all() and torch.isnan(lse[0, 0, 1])
    x = f64(kv[0])
    x[n - 1] = 0
    seen = oracle.visible(M, n)
    for h in sorted({0, H - 1}):
        rest = [m for m in range(M - 1) if (m, h) != (1, 0)]
        ref = oracle.attention(f64(q[0, rest, h]), x, x[:, :dc], 0.05, [seen[m] for m in rest])
        check(out[:, rest], lse[:, :, rest], 0, h, ref, 288, dtype, n, np.abs(x).max())
        assert torch.isnan(out[0, M - 1, h, 4].float())
        keep = [c for c in range(dc) if c != 4]
        ref = oracle.attention(f64(q[0, M - 1:, h]), x, x[:, :dc], 0.05, [seen[M - 1][:-1]])
        ref = {**ref, "out": ref["out"][:, keep], "mass": ref["mass"][:, keep]}
        check(out[:, M - 1:][..., keep], lse[:, :, M - 1:], 0, h, ref, 288, dtype, n, np.abs(x).max())


@pytest.mark.parametrize("dtype", [BF, F16, F32])
@pytest.mark.parametrize("M,causal", [(1, True), (7, False), (7, True), (40, False)])
@pytest.mark.parametrize("n", [70, 64, 129])
def test_expanded_infinite_last_value(gpu, dtype, M, causal, n):
    """The last key stands in for those behind it in its tile, with no weight: its infinite value is infinite for the rows
    that see it, in its own column, and stays out of the others."""
    q, k, pe, v, sl = make_exp(dtype, 1, M, 150, 2, 64, 32, [n], seed=M)
    v[0, n - 1, 0, 9] = math.inf
    out, lse = latent_attn_expanded(q, k, pe, v, cache_seqlens=sl, causal=causal, return_softmax_lse=True)
    seen = oracle.visible(M, n, causal=causal)
    hit = [m for m in range(M) if n - 1 in seen[m]]
    assert torch.equal(out[0, hit, 0, 9].float(), torch.full((len(hit),), math.inf, device=gpu))
    for h in range(2):
        x, y = np.concatenate([f64(k[0, :n, h]), f64(pe[0, :n])], -1), f64(v[0, :n, h])
        y[n - 1, 9] = 0.0 if h == 0 else y[n - 1, 9]
        ref = oracle.attention(f64(q[0, :, h]), x, y, 96 ** -0.5, seen)
        got = out.clone()
        if h == 0:
            got[0, hit, 0, 9] = torch.from_numpy(ref["out"][hit, 9]).to(got)
        check(got, lse, 0, h, ref, 96, dtype, n, np.abs(y).max())
