"""Expanded latent attention: what the exponents' common offset rounds away."""

import math

import numpy as np
import pytest
import torch

from diffspec_mi355x.runtime.latent_attention import latent_attn_expanded
from test_gpu_latent import BF, F16, F32, f64

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [BF, F16, F32])
@pytest.mark.parametrize("top", [1453637, 1453636, 1453633, 1453629, 726820, 726812, 11, 0])
@pytest.mark.parametrize("M", [1, 40])
def test_a_later_maximum_of_scores_far_below_zero(gpu, dtype, top, M):
    """32 keys of a score of -top (in units of log2 within 10 of 2^21 and of 2^20, where an offset added to the maximum
    rounds by up to 1/8), then one of 4 more, which moves the maximum.

    Scores are sums of two products of short numbers, exact in fp32.  Bounds of weights: those of test_gpu_latent.py with
    delta 0, the product of a difference of up to 4 with the scale (2^-23 of it) in its place."""
    n = 64 + M - 1
    k = torch.zeros((1, n, 1, 64), dtype=torch.float64)
    big = top // 1024 if dtype != BF else top // 1024 // 8 * 8  # (bf16: eight bits)
    rest = top - 1024 * big
    a, b, c = (rest // 64, rest % 64, 1)
    k[0, :, 0, 0] = -big
    k[0, :, 0, 1] = -a
    k[0, :, 0, 2] = -b
    k[0, 32:, 0, 3] = -200
    k[0, 40, 0, 3] = 4
    q = torch.zeros((1, M, 1, 96), dtype=torch.float64)
    q[..., 0], q[..., 1], q[..., 2], q[..., 3] = 1024, 64, 1, c
    g = torch.Generator().manual_seed(top)
    v = torch.randn((1, n, 1, 64), generator=g)
    k, q, v = (x.to(dtype).to(gpu) for x in (k, q, v))
    pe = torch.zeros((1, n, 32), dtype=dtype, device=gpu)
    x, y = f64(k[0, :, 0]), f64(v[0, :, 0])
    s = x[:, :4] @ np.array([1024.0, 64.0, 1.0, c])
    assert s[0] == -top and s[40] == 4 - top
    out, lse = latent_attn_expanded(q, k, pe, v, softmax_scale=1.0, return_softmax_lse=True)
    u = 0.0 if dtype == F32 else torch.finfo(dtype).eps / 2
    for m in range(M):
        e = 64 + m
        w = np.exp(s[:e] - s[:e].max())
        ref, mass = (w @ y[:e]) / w.sum(), (w @ np.abs(y[:e])) / w.sum()
        tol = mass * (u + 8 * 2.0 ** -24 + (e + 64) * 2.0 ** -24 + 2.0 ** -22) * 1.01 + torch.finfo(dtype).eps / 2 * np.abs(ref)
        tol = tol + e * 2.0 ** -34 * np.abs(y).max()
        assert (np.abs(f64(out[0, m, 0]) - ref) <= tol).all(), m
        want = s[:e].max() + math.log(w.sum())
        assert abs(float(lse[0, 0, m]) - want) <= 2.0 ** -22 * abs(want) + (e + 64) * 2.0 ** -24 + 2.0 ** -22
