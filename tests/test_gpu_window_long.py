"""Windowed attention over long windows: probabilities below fp16's range."""

import numpy as np
import pytest
import torch

from diffspec_mi355x.runtime.window_attention import window_attn_with_kvcache
from test_gpu_window import F16

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("gap", [10.0, 14.0, 16.0, 17.5, 18.5])
@pytest.mark.parametrize("M", [1, 40])
def test_f16_many_small_probabilities(gpu, M, gap):
    """One key ``gap`` above 2^18 others, whose probabilities lie below fp16's range but whose sum does not; sequences
    enough (all of the same keys) that no key range is shared out.

    Relative to the running maximum a probability is rounded to fp16 after a
    factor of 2^10 at least: off by 2^-11 of itself or, below 2^-24, by 2^-35.
    Sums: an accumulator takes 16 keys at a time, so n / 16 fp32 roundings; the
    scores are exact but for the exponent's argument and the exponential, 2^-21
    and (D + 4) 2^-24 of the score.
    """
    B, N, D = 300, 1 << 18, 64
    g = torch.Generator().manual_seed(M)
    q = torch.ones((B, M, 1, D), dtype=F16, device=gpu)
    k = torch.zeros((1, N, 1, D), dtype=F16, device=gpu)
    k[0, 3] = gap / 8.0
    gap = float(k[0, 3, 0, 0]) * 8.0
    v = torch.rand((1, N, 1, D), generator=g).to(F16).to(gpu)
    v[0, 3] = 0.0
    out, lse = window_attn_with_kvcache(q, k.expand(B, -1, -1, -1), v.expand(B, -1, -1, -1), N + 1, 0, return_softmax_lse=True)
    assert bool((out == out[:1]).all()) and bool((lse == lse[:1]).all())
    total = v[0, :, 0].double().cumsum(0).cpu().numpy()
    for m in range(M):
        n = N - M + m + 1
        z = 1.0 + (n - 1) * np.exp(-gap)
        want = total[n - 1] * np.exp(-gap) / z
        rel = 2 * ((D + 4) * 2.0 ** -24 * gap + 2.0 ** -21) + 2 * (n / 16 + 64) * 2.0 ** -24
        tol = want * (rel + 2.0 ** -11 + 1.01 * 2.0 ** -11) + n * 2.0 ** -35 + 2.0 ** -25
        assert (np.abs(out[0, m, 0].double().cpu().numpy() - want) <= tol).all(), (m, out[0, m, 0, :2], want[:2], tol[:2])
        assert abs(float(lse[0, 0, m]) - (gap + np.log(z))) <= rel + 2.0 ** -22 * (1 + gap)
