"""Windowed attention over long windows: keys shared out over workgroups, scores that outgrow the running maximum,
probabilities below fp16's range, hidden values behind a split."""

import numpy as np
import pytest
import torch

from diffspec_mi355x import _ext, workloads as wl
from diffspec_mi355x.runtime.window_attention import window_attn_with_kvcache
from oracle import window as oracle
from test_gpu_window import BF16, F16, F32, Case

pytestmark = pytest.mark.gpu


def shared_out(lib, c, window, sinks, tree=False):
    """Does the call share the keys out over workgroups (and so need a workspace)?"""
    H, D = c.q.shape[2:]
    Hk = c.k.shape[2 if c.table is None else 1]
    cap = c.k.shape[1] if c.table is None else c.table.shape[1] * c.page
    return lib.dsv_window_workspace_bytes(c.B, c.M, H, Hk, D, _ext.desc(c.q).dtype, cap, window, sinks, int(tree)) > 0


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("B,M,H,Hk,D,lens,window,sinks,page", [
    (1, 1, 1, 1, 64, [1500], 1400, 0, 0),
    (1, 1, 8, 2, 128, [3000], 2900, 40, 16),
    (2, 1, 32, 8, 128, [5000, 1300], 4096, 4, 64),
    (3, 1, 14, 2, 64, [4000, 0, 37], 2048, 33, 8),
    (1, 2, 8, 1, 64, [2500], 5000, 0, 4),
    (1, 5, 6, 2, 64, [3001], 2800, 70, 1),
    (2, 16, 2, 2, 128, [2700, 1400], 2500, 1, 0)])
def test_few_rows_shared_out(gpu, dsv_lib, B, M, H, Hk, D, lens, window, sinks, page, dtype):
    c = Case(gpu, B, M, H, Hk, D, lens, dtype, page, seed=M + H)
    assert shared_out(dsv_lib, c, window, sinks)
    c.check(window, sinks)


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("M,H,Hk,D,page", [(8, 4, 2, 64, 16), (16, 1, 1, 128, 0), (5, 6, 2, 128, 32)])
def test_small_trees_shared_out(gpu, dsv_lib, M, H, Hk, D, page, dtype):
    lens, window, sinks = [2600, 2300], 2200, 20
    c = Case(gpu, 2, M, H, Hk, D, lens, dtype, page, seed=M)
    assert shared_out(dsv_lib, c, window, sinks, True)
    c.check(window, sinks, [wl.make_tree(M, max_depth=M, max_outdeg=3, seed=M + i)[0] for i in range(2)])


@pytest.mark.parametrize("M,H,Hk,D,page", [(40, 4, 2, 64, 16), (70, 2, 1, 128, 0)])
def test_many_fp32_rows_shared_out(gpu, dsv_lib, M, H, Hk, D, page):
    c = Case(gpu, 1, M, H, Hk, D, [2500], F32, page, seed=M)
    assert shared_out(dsv_lib, c, 2200, 20)
    c.check(2200, 20)


def ramp(c, per_tile):
    """Keys whose scores change by about per_tile (natural log units) from a tile of 32 to the next."""
    N, D = c.k.shape[1], c.k.shape[3]
    c.q[:] = 1.0
    level = torch.arange(N, device=c.gpu).double() * (per_tile / 32) / (D ** 0.5)
    level -= level.mean()
    c.k.copy_((level.view(1, N, 1, 1) + 0.02 * c.k.double()).to(c.k.dtype))


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("per_tile", [-20.0, -1.0, 0.6, 3.0, 7.0, 20.0])
@pytest.mark.parametrize("M,H,D", [(200, 2, 64), (40, 2, 128), (3, 2, 64)])
def test_scores_that_grow(gpu, dtype, per_tile, M, H, D):
    """Scores that outgrow (or fall behind) the running maximum in every tile, masked and unmasked ones."""
    c = Case(gpu, 1, M, H, 1, D, [1700], dtype, 0, seed=M)
    ramp(c, per_tile)
    c.check(1400, 5)
    if M == 200:  # (blocks enough that no key range is shared out)
        c = Case(gpu, 64, 20, 16, 4, D, [1100] * 64, dtype, 0, seed=M)
        ramp(c, per_tile)
        out = window_attn_with_kvcache(c.q, c.k, c.v, 1000, 5, return_softmax_lse=True)
        c.B, c.lens = 1, [1100]
        c.check(1000, 5, result=out)


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("M", [2, 150])
def test_large_scores(gpu, dtype, M):
    """Scores of deviation 30 through long unmasked stretches."""
    Case(gpu, 1, M, 4, 2, 128, [1500], dtype, 16, seed=8, scale=30.0).check(1300, 4)


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


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("M,G", [(4, 2), (16, 1), (40, 2)])
def test_hidden_values_shared_out(gpu, dsv_lib, M, G, dtype):
    """An infinite or NaN entry of V reaches the rows that see its key and no others, where the keys are shared out."""
    n, window, sinks = 2600, 2200, 2
    c = Case(gpu, 1, M, 2 * G, 2, 64, [n], dtype, 0, seed=3)
    assert shared_out(dsv_lib, c, window, sinks)
    keys = oracle.visible(M, n, window, sinks)
    clean = c.v.clone()
    c.v[0, :, 0] = clean[0, :, 0]
    for key in (n - M - window + 2, n - M // 2, n - 1):
        for kind in (float("inf"), float("nan")):
            c.v[0, key, 1, 5] = kind
            out = window_attn_with_kvcache(c.q, c.k, c.v, window, sinks, return_softmax_lse=True)
            sees = torch.tensor([key in x for x in keys], device=gpu)
            assert bool(sees.any())
            assert torch.equal(~torch.isfinite(out[0][0, :, G:, 5]).any(-1), sees), (key, kind)
            # The rows and columns that it does not reach, against the other values' sums.
            c.v.copy_(clean)
            fixed = out[0].clone()
            ref = window_attn_with_kvcache(c.q, c.k, c.v, window, sinks)
            fixed[0, sees, G:, 5] = ref[0, sees, G:, 5]
            c.check(window, sinks, result=(fixed, out[1]))


@pytest.mark.parametrize("dtype", [BF16, F16])
def test_hidden_tree_values_shared_out(gpu, dsv_lib, dtype):
    """The same for siblings of a tree over a long prefix."""
    M, n, window, sinks = 30, 2600, 2200, 2
    parent = wl.make_tree(M, max_depth=M, max_outdeg=3, seed=4)[0]
    c = Case(gpu, 1, M, 4, 2, 64, [n], dtype, 16, seed=4)
    assert shared_out(dsv_lib, c, window, sinks, True)
    keys = oracle.visible(M, n, window, sinks, parent)
    par = torch.tensor(parent, device=gpu)
    slot = c.slot(c.v, 0, n - 3)
    good = slot.clone()
    slot[1, 7] = float("inf")
    out = window_attn_with_kvcache(c.q, c.k, c.v, window, sinks, n, c.table, par, True)
    slot.copy_(good)
    ref = window_attn_with_kvcache(c.q, c.k, c.v, window, sinks, n, c.table, par)
    sees = torch.tensor([n - 3 in x for x in keys], device=gpu)
    assert torch.equal(~torch.isfinite(out[0][0, :, 2:, 7]).any(-1), sees)
    fixed = out[0].clone()
    fixed[0, sees, 2:, 7] = ref[0, sees, 2:, 7]
    c.check(window, sinks, parent, result=(fixed, out[1]))


@pytest.mark.parametrize("M", [1, 40])
@pytest.mark.parametrize("huge", [(1 << 63) - 1, 1 << 63, (1 << 64) + 9, 10 ** 30])
def test_windows_beyond_64_bits(gpu, huge, M):
    """A window or sinks beyond every key mean all of them, however large the number."""
    c = Case(gpu, 2, M, 8, 2, 64, [1500, 1500], BF16, 16, seed=M)
    want = c.check(1500, 0)
    for window, sinks in ((huge, 0), (1, huge)):
        got = window_attn_with_kvcache(c.q, c.k, c.v, window, sinks, 1500, c.table, None, True)
        assert torch.allclose(got[0].float(), want[0].float(), rtol=2 ** -6, atol=2 ** -6)
        c.check(1500, 0, result=got)
    with pytest.raises(RuntimeError):
        window_attn_with_kvcache(c.q, c.k, c.v, -huge, 0, 1500, c.table)


@pytest.mark.parametrize("dtype,power", [(F16, 9), (F16, 11), (F16, 12), (F16, 13), (F16, 15), (BF16, 11), (BF16, 13), (BF16, 16),
                                         (BF16, 20), (BF16, 40), (F32, 11), (F32, 13), (F32, 16), (F32, 20), (F32, 40)])
@pytest.mark.parametrize("level", [0.25, 0.2744140625, 0.3056640625, 0.33203125])
@pytest.mark.parametrize("M,H,B", [(1, 2, 1), (3, 2, 150), (40, 1, 1), (200, 1, 1), (20, 1, 260)])
def test_scores_beyond_the_exponents_resolution(gpu, dtype, power, level, M, H, B):
    """Scores around 2^(2 power + 1), whose product with the exponent's scale is off by more than a probability may be.

    One key's score is twice the next one's, so its value is the output: off by
    the rounding of its probability and the output's own; the score is exact (equal
    powers of two, eight bits of level) and the log-sum-exp two fp32 products of it.
    """
    N, D, window = 1500, 64, 1200
    g = torch.Generator().manual_seed(power)
    sign = torch.where(torch.rand((1, 1, H, 1), generator=g) < 0.5, -1.0, 1.0)
    q = (2.0 ** power * sign).expand(B, M, H, D).to(dtype).to(gpu)
    k = torch.zeros((1, N, H, D), dtype=dtype)
    top = N - M - 40
    for n, f in ((top - 900, level / 4), (top - 500, level / 2), (top, level)):
        k[0, n] = (f * 2.0 ** power * sign[0, 0]).expand(H, D).to(dtype)
    v = torch.randn((1, N, H, D), generator=g).to(dtype)
    k, v = k.to(gpu), v.to(gpu)
    out, lse = window_attn_with_kvcache(q, k.expand(B, -1, -1, -1), v.expand(B, -1, -1, -1), window, 0, return_softmax_lse=True)
    want = v[0, top].double().expand(B, M, H, D)
    step = 0.0 if dtype == F32 else torch.finfo(dtype).eps / 2
    assert bool(((out.double() - want).abs() <= want.abs() * (2.02 * step + 2.0 ** -20)).all())
    score = float((q[0, 0, 0].double() * k[0, top, 0].double()).sum()) / D ** 0.5
    assert bool(((lse.double() - score).abs() <= score * 2.0 ** -21).all())
