"""Absorbed latent attention of very many sequences: the time grows with them, not with their square."""

import math

import numpy as np
import pytest
import torch

from diffspec_mi355x.runtime.latent_attention import latent_attn_with_kvcache
from oracle import latent as oracle
from test_gpu_latent import BF, F32, check, f64

pytestmark = pytest.mark.gpu


def inputs(dtype, B, H, N):
    g = torch.Generator(device="cuda").manual_seed(B)
    kv = torch.randn((B, N, 288), generator=g, device="cuda", dtype=dtype)
    q = torch.randn((B, 1, H, 288), generator=g, device="cuda", dtype=dtype)
    lens = torch.randint(0, N + 1, (B,), generator=g, device="cuda", dtype=torch.int32)
    return q, kv, lens


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("B,H,N", [(70000, 1, 4), (5000, 3, 130), (300, 2, 1000), (255, 16, 70), (256, 16, 70), (257, 16, 70), (258, 16, 70)])
def test_cut_sequences_are_joined(gpu, dtype, B, H, N):
    q, kv, lens = inputs(dtype, B, H, N)
    out, lse = latent_attn_with_kvcache(q, kv, 256, 0.06, cache_seqlens=lens, return_softmax_lse=True)
    n = lens.tolist()
    # Whole batches in torch's float32 (its error is that of the kernel's scores), some in float64.
    keep = torch.arange(N, device=gpu)[None, :] < lens[:, None]
    for lo in range(0, B, 1000):
        hi = min(B, lo + 1000)
        s = torch.matmul(q[lo:hi, 0].float(), kv[lo:hi].float().transpose(1, 2).contiguous()) * 0.06
        s = s.masked_fill(~keep[lo:hi, None], -math.inf)
        p = torch.nan_to_num(torch.softmax(s, -1), nan=0.0)
        want = torch.matmul(p, kv[lo:hi, :, :256].float())
        # (Weights and output rounded to 8 bits, values up to 6: far above what a cut sequence left out would show.)
        assert (out[lo:hi, 0].float() - want).abs().max() <= 6 * 2.0 ** -7, lo
        assert torch.equal(torch.isneginf(lse[lo:hi, :, 0]), (lens[lo:hi] == 0)[:, None].expand(hi - lo, H)), lo
    rng = np.random.default_rng(B)
    for b in sorted({0, B - 1, *(int(x) for x in rng.integers(0, B, 40))}):
        x = f64(kv[b, :n[b]])
        for h in range(H):
            ref = oracle.attention(f64(q[b, :, h]), x, x[:, :256], 0.06, oracle.visible(1, n[b]))
            check(out, lse, b, h, ref, 288, dtype, max(n[b], 1), np.abs(x).max() if n[b] else 0.0)


def test_time_grows_with_the_batch(gpu):
    """Four times the sequences take about four times the time (16 times if each were sought among all)."""
    took = []
    for B in (1 << 15, 1 << 17):
        q, kv, lens = inputs(BF, B, 1, 4)
        call = lambda: latent_attn_with_kvcache(q, kv, 256, 0.06, cache_seqlens=lens)  # noqa: E731
        call()
        best = math.inf
        for _ in range(5):
            a, b = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
            a.record()
            call()
            b.record()
            torch.cuda.synchronize()
            best = min(best, a.elapsed_time(b))
        took.append(best)
    print("ms:", took)
    assert took[1] <= 8 * took[0], took
