"""Latent attention (absorbed and expanded) against the float64 oracle.

Error bounds, for u half a step of the 16-bit type, D the width of a score's sum, n the
keys of a row (scores and sums are fp32, half a step 2^-24):
  scores    a sum of D products in any order is off by D 2^-24 sum |q k|, scaled:
            delta = (D + 2) 2^-24 reach, so weights by a factor e^(2 delta) at most;
  weights   rounded to 16 bits: u each (fp16 holds them times 2^10, so what it flushes is
            below 2^-34 of the largest: n 2^-34 max|v| in all); exp2 itself 2^-22;
  sums      n + 64 additions (pieces, waves and splits among them): (n + 64) 2^-24;
  output    rounded once more: u |out|.
All but the last two apply to the weighted mean of |v| ("mass").  lse: delta, the sum's
(n + 64) 2^-24 + 2^-22, and 2^-22 |lse| for its own rounding.
"""

import math

import numpy as np
import pytest
import torch

from diffspec_mi355x.runtime.latent_attention import latent_attn_expanded, latent_attn_with_kvcache
from oracle import latent as oracle

pytestmark = pytest.mark.gpu

BF, F16, F32 = torch.bfloat16, torch.float16, torch.float32


def f64(t):
    return t.detach().double().cpu().numpy()


def check(out, lse, b, h, ref, D, dtype, n, vmax):
    u = torch.finfo(out.dtype).eps / 2
    up = 0.0 if dtype == F32 else torch.finfo(dtype).eps / 2
    delta = (D + 2) * 2.0 ** -24 * ref["reach"][:, None]
    tail = (n + 64) * 2.0 ** -24 + 2.0 ** -22
    tol = ref["mass"] * (np.expm1(2 * delta) + up + tail) * 1.01 + u * np.abs(ref["out"]) + n * 2.0 ** -34 * vmax + 1e-30
    got = f64(out[b, :, h])
    bad = ~(np.abs(got - ref["out"]) <= tol)
    assert not bad.any(), (b, h, np.argwhere(bad)[:3], np.abs(got - ref["out"])[bad][:3], tol[bad][:3])
    if lse is not None:
        gl, rl = f64(lse[b, h]), ref["lse"]
        assert np.array_equal(np.isneginf(gl), np.isneginf(rl)), (b, h)
        ok = np.isfinite(rl)
        lt = delta[:, 0] + tail + 2.0 ** -22 * np.abs(np.where(ok, rl, 0))
        assert (np.abs(gl - rl)[ok] <= lt[ok]).all(), (b, h, np.abs(gl - rl)[ok].max())


def chain_tree(rng, M):
    return [-1] + [int(rng.integers(max(0, i - 6), i)) for i in range(1, M)]


def make(dtype, B, M, H, dc, dr, page, lens, tree, seed=0, table_dtype=torch.int32, spare=5, scale=1.0):
    """Inputs whose unseen places (behind the lengths, unused pages) hold NaN and whose table entries there are -1."""
    rng = np.random.default_rng(seed)
    g = torch.Generator(device="cuda").manual_seed(seed)
    D, N = dc + dr, max(max(lens), 1)
    rows = [torch.randn((n, D), generator=g, device="cuda").to(dtype) for n in lens]
    if page:
        need = [-(-n // page) for n in lens]
        P = sum(need) + spare
        ids = rng.permutation(P)
        kv = torch.full((P, page, D), math.nan, dtype=dtype, device="cuda")
        table = torch.full((B, -(-N // page) + 1), -1, dtype=table_dtype)
        at = 0
        for b, (k, x) in enumerate(zip(need, rows)):
            pg = torch.from_numpy(ids[at:at + k])
            table[b, :k] = pg.to(table_dtype)
            pad = torch.full((k * page, D), math.nan, dtype=dtype, device="cuda")
            pad[:lens[b]] = x
            kv[pg.cuda()] = pad.view(k, page, D)
            at += k
        table = table.cuda()
    else:
        table = None
        kv = torch.full((B, N, D), math.nan, dtype=dtype, device="cuda")
        for b, x in enumerate(rows):
            kv[b, :lens[b]] = x
    q = (torch.randn((B, M, H, D), generator=g, device="cuda") * scale).to(dtype)
    parent = None
    if tree:
        parent = torch.tensor([chain_tree(rng, M) for _ in range(B)], dtype=torch.int32, device="cuda")
    return q, kv, table, torch.tensor(lens, dtype=torch.int32, device="cuda"), parent, rows


def compare(q, rows, lens, dc, scale, out, lse, parent, heads, dtype):
    M = q.shape[1]
    for b, n in enumerate(lens):
        x = f64(rows[b])
        seen = oracle.visible(M, n, None if parent is None else parent[b].tolist())
        vmax = np.abs(x).max() if n else 0.0
        for h in heads:
            ref = oracle.attention(f64(q[b, :, h]), x, x[:, :dc], scale, seen)
            check(out, lse, b, h, ref, q.shape[3], dtype, n, vmax)


CASES = [
    # dtype, B, M, H, dc, dr, page, lens, tree
    (BF, 1, 1, 16, 512, 64, 64, [1], False),
    (BF, 1, 1, 128, 512, 64, 64, [2900], False),
    (BF, 5, 1, 16, 512, 64, 16, [0, 1, 63, 64, 65], False),
    (F16, 5, 1, 16, 512, 64, 16, [0, 1, 63, 640, 1000], False),
    (F32, 5, 1, 16, 512, 64, 16, [0, 1, 63, 64, 65], False),
    (BF, 3, 1, 20, 512, 32, 8, [700, 5, 129], False),
    (F16, 3, 1, 33, 256, 64, 0, [700, 5, 129], False),
    (BF, 3, 1, 128, 256, 32, 1, [70, 300, 129], False),
    (F32, 3, 1, 128, 256, 32, 2, [70, 300, 129], False),
    (BF, 2, 7, 8, 512, 64, 32, [3, 500], False),
    (F16, 2, 130, 3, 512, 64, 128, [130, 64], False),
    (F32, 2, 37, 3, 256, 64, 4, [37, 200], False),
    (BF, 2, 200, 1, 512, 64, 16, [200, 1111], False),
    (BF, 3, 64, 16, 512, 64, 16, [64, 1500, 40], True),
    (F16, 2, 33, 5, 256, 32, 64, [400, 33], True),
    (F32, 2, 33, 5, 512, 32, 0, [400, 20], True),
    (BF, 1, 700, 1, 512, 64, 64, [900], True),
    (BF, 1, 1024, 2, 256, 64, 0, [1100], True),
    (F32, 1, 700, 1, 256, 64, 64, [750], True),
    (BF, 40, 1, 16, 512, 64, 64, [(i * 97) % 700 for i in range(40)], False),
]


@pytest.mark.parametrize("dtype,B,M,H,dc,dr,page,lens,tree", CASES)
def test_absorbed(gpu, dtype, B, M, H, dc, dr, page, lens, tree):
    q, kv, table, sl, parent, rows = make(dtype, B, M, H, dc, dr, page, lens, tree, seed=M + H)
    scale = 1.7 / math.sqrt(dc + dr)
    out, lse = latent_attn_with_kvcache(q, kv, dc, scale, cache_seqlens=sl, page_table=table, parent=parent,
                                        return_softmax_lse=True)
    torch.cuda.synchronize()
    assert out.shape == (B, M, H, dc) and out.dtype == dtype and lse.shape == (B, H, M)
    heads = range(H) if B * M * H <= 256 else sorted({0, H // 2, H - 1})
    compare(q, rows, lens, dc, scale, out, lse, parent, heads, dtype)


@pytest.mark.parametrize("dtype", [BF, F16])
@pytest.mark.parametrize("H", [1, 16, 17, 32, 48, 64, 65])
def test_absorbed_row_blocks_and_splits(gpu, dtype, H):
    """Every block size, and sequences that many workgroups share."""
    lens = [9000, 3, 4097]
    q, kv, table, sl, _, rows = make(dtype, 3, 1, H, 512, 64, 32, lens, False, seed=H)
    out, lse = latent_attn_with_kvcache(q, kv, 512, 0.05, cache_seqlens=sl, page_table=table, return_softmax_lse=True)
    compare(q, rows, lens, 512, 0.05, out, lse, None, sorted({0, H // 3, H - 1}), dtype)


@pytest.mark.parametrize("dtype", [BF, F16, F32])
def test_absorbed_layouts(gpu, dtype):
    """Strided q, cache rows and outputs, int64 and shared tables, scalar lengths, other output types."""
    B, M, H, dc, dr, page, n = 3, 4, 6, 256, 64, 16, 150
    q, kv, table, sl, _, rows = make(dtype, 1, M, H, dc, dr, page, [n], False, seed=1, table_dtype=torch.int64)
    wide = torch.zeros((B, H, M, dc + dr + 16), dtype=dtype, device=gpu)
    qs = wide[..., 8:8 + dc + dr].transpose(1, 2)
    qs.copy_(q.expand(B, M, H, dc + dr))
    pool = torch.full((kv.shape[0], 2, page, dc + dr + 24), math.nan, dtype=dtype, device=gpu)
    pool[:, 1, :, :dc + dr] = kv
    for od in (BF, F16, F32):
        out, lse = latent_attn_with_kvcache(qs, pool[:, 1, :, :dc + dr], dc, 0.06, cache_seqlens=n, page_table=table[0],
                                            return_softmax_lse=True, out_dtype=od)
        assert out.dtype == od
        compare(qs, rows * B, [n] * B, dc, 0.06, out, lse, None, range(H), dtype)
    again = latent_attn_with_kvcache(qs, pool[:, 1, :, :dc + dr], dc, 0.06, cache_seqlens=torch.full((B,), n + 10 ** 6, device=gpu),
                                     page_table=table[:, :10].contiguous())
    # (the lengths are clamped to the table: 10 pages)
    seen10 = [160] * B
    full = pool[:, 1, :, :dc + dr][table[0, :10].clamp(min=0)].reshape(160, -1)
    if not torch.isnan(full).any():
        compare(qs, [full] * B, seen10, dc, 0.06, again, None, None, range(H), dtype)


@pytest.mark.parametrize("dtype", [BF, F16, F32])
@pytest.mark.parametrize("tree", [False, True])
def test_absorbed_hidden_values(gpu, dtype, tree):
    """Infinite and NaN rows of tokens that only some queries see reach those alone."""
    M, H, n = 24, 5, 300
    q, kv, _, sl, parent, rows = make(dtype, 2, M, H, 512, 64, 0, [n, n], tree, seed=3)
    kv[0, n - 1, 7] = math.inf
    kv[1, n - 5, 3] = math.nan
    kv[1, n - 5, 540] = 1.0
    out, lse = latent_attn_with_kvcache(q, kv, 512, 0.05, cache_seqlens=sl, parent=parent, return_softmax_lse=True)
    for b, hit in ((0, n - 1), (1, n - 5)):
        x = f64(kv[b])
        seen = oracle.visible(M, n, parent[b].tolist() if tree else None)
        clean = [m for m in range(M) if hit not in seen[m]]
        assert clean and len(clean) < M
        x[hit] = 0
        for h in range(H):
            ref = oracle.attention(f64(q[b, clean, h]), x, x[:, :512], 0.05, [seen[m] for m in clean])
            check(out[:, clean], lse[:, :, clean], b, h, ref, 576, dtype, n, np.abs(x).max())
        dirty = [m for m in range(M) if hit in seen[m]]
        assert not torch.isfinite(out[b, dirty].float()).all(-1).any()


@pytest.mark.parametrize("dtype", [BF, F16, F32])
@pytest.mark.parametrize("H,M,n", [(128, 5, 70), (64, 3, 9000), (16, 9, 200), (48, 4, 130)])
def test_absorbed_hidden_siblings(gpu, dtype, H, M, n):
    """Blocks of rows that all belong to one node of a tree: its siblings' infinite and NaN rows stay out of them."""
    q, kv, _, sl, _, rows = make(dtype, 1, M, H, 512, 64, 0, [n], False, seed=H)
    parent = torch.tensor([-1] + [0] * (M - 1), dtype=torch.int32, device=gpu)  # (a root and its children)
    kv[0, n - 1, 7] = math.inf      # the last child
    kv[0, n - M + 1, 3] = math.nan  # the first
    out, lse = latent_attn_with_kvcache(q, kv, 512, 0.05, cache_seqlens=sl, parent=parent, return_softmax_lse=True)
    x = f64(kv[0])
    seen = oracle.visible(M, n, parent.tolist())
    clean = [m for m in range(M) if m not in (1, M - 1)]
    x[n - 1] = x[n - M + 1] = 0
    for h in (0, H // 2, H - 1):
        ref = oracle.attention(f64(q[0, clean, h]), x, x[:, :512], 0.05, [seen[m] for m in clean])
        check(out[:, clean], lse[:, :, clean], 0, h, ref, 576, dtype, n, np.abs(x).max())
    assert not torch.isfinite(out[0, 1].float()).all(-1).any() and not torch.isfinite(out[0, M - 1].float()[:, 7]).any()


@pytest.mark.parametrize("dtype", [BF, F16, F32])
@pytest.mark.parametrize("H", [8, 33, 64])
def test_absorbed_infinite_last_value(gpu, dtype, H):
    """An infinite entry of the last token, which stands in for those behind it in its tile: a score of 0 * inf spoils the
    row, one of -inf (no weight) its own column alone."""
    n = 90
    q, kv, _, sl, _, rows = make(dtype, 1, 1, H, 256, 32, 0, [n], False, seed=H)
    q[..., 9] = 0
    kv[0, n - 1, 9] = math.inf
    out, lse = latent_attn_with_kvcache(q, kv, 256, 0.05, cache_seqlens=sl, return_softmax_lse=True)
    assert torch.isnan(out.float()).all() and torch.isnan(lse).all()
    q[..., 9] = -2.0 ** -14
    out, lse = latent_attn_with_kvcache(q, kv, 256, 0.05, cache_seqlens=sl, return_softmax_lse=True)
    assert torch.isnan(out[..., 9].float()).all()  # (0 * inf, as the formula has it)
    keep = [c for c in range(256) if c != 9]
    x = f64(kv[0, :n - 1])
    for h in range(H):
        ref = oracle.attention(f64(q[0, :, h]), x, x[:, :256], 0.05, [np.arange(n - 1)])  # (x holds no infinity)
        ref = {**ref, "out": ref["out"][:, keep], "mass": ref["mass"][:, keep]}
        check(out[..., keep], lse, 0, h, ref, 288, dtype, n, np.abs(x).max())


@pytest.mark.parametrize("dtype", [BF, F16, F32])
@pytest.mark.parametrize("size", [30.0, 3e3, 1e6])
def test_absorbed_large_and_growing_scores(gpu, dtype, size):
    """Scores that grow along the cache, so that the maximum moves in every tile, up to far beyond 2^22."""
    if dtype == F16 and size > 1e4:
        size = 2e4
    n, H, dc = 900, 16, 256
    kv = torch.zeros((1, n, dc + 32), dtype=dtype, device=gpu)
    kv[0, :, 0] = (torch.arange(n, device=gpu) // 3 * 0.25).to(dtype)
    kv[0, :, 1:dc] = torch.randn((n, dc - 1), device=gpu).to(dtype)
    q = torch.zeros((1, 1, H, dc + 32), dtype=dtype, device=gpu)
    q[..., 0] = (torch.linspace(0.01, 1, H, device=gpu) * size).to(dtype)
    out, lse = latent_attn_with_kvcache(q, kv, dc, 0.7, return_softmax_lse=True)
    # Scores of one product, exact in fp32 but for their rounding: weights of equal rows are exact.
    x = f64(kv[0])
    for h in range(H):
        s = np.float32(f64(q[0, 0, h, 0])) * np.float32(x[:, 0])
        w = np.exp((s.astype(np.float64) - float(s.max())) * 0.7)
        ref = (w[:, None] * x[:, :dc]).sum(0) / w.sum()
        mass = (w[:, None] * np.abs(x[:, :dc])).sum(0) / w.sum()
        u = torch.finfo(dtype).eps
        # differences of scores are exact near the maximum; their product with the scale is off by 2^-24 of up to 40
        tol = mass * (u + 80 * 2.0 ** -24 + (n + 64) * 2.0 ** -24) + 1e-6
        assert (np.abs(f64(out[0, 0, h]) - ref) <= tol).all(), h
        want = float(s.max()) * 0.7 + math.log(w.sum())
        assert abs(float(lse[0, h, 0]) - want) <= 1e-5 + 2.0 ** -21 * abs(want)


def test_absorbed_infinite_scores(gpu):
    q, kv, _, sl, _, rows = make(BF, 1, 1, 16, 512, 64, 0, [200], False, seed=9)
    kv[0, 50, 515] = -math.inf
    q[..., 515] = q[..., 515].abs() + 0.1
    out, lse = latent_attn_with_kvcache(q, kv, 512, 0.05, return_softmax_lse=True)
    keep = [i for i in range(200) if i != 50]
    x = f64(kv[0, keep])
    for h in range(16):
        ref = oracle.attention(f64(q[0, :, h]), x, x[:, :512], 0.05, [np.arange(199)])
        check(out, lse, 0, h, ref, 576, BF, 200, np.abs(x[:, :512]).max())
    kv[0, :, 515] = -math.inf  # no finite score: no key
    out, lse = latent_attn_with_kvcache(q, kv, 512, 0.05, return_softmax_lse=True)
    assert (out == 0).all() and torch.isneginf(lse).all()


def test_absorbed_far_pages(gpu):
    """Pages whose byte offsets pass 2^32."""
    page, D = 64, 576
    P = (9 << 30) // (page * D * 2)
    pool = torch.empty((P, page, D), dtype=BF, device=gpu)
    ids = torch.tensor([P - 1, 3, P // 2 + 1, P - 7], device=gpu)
    pool[ids] = torch.randn((4, page, D), device=gpu).to(BF)
    q = torch.randn((1, 1, 16, D), device=gpu).to(BF)
    out, lse = latent_attn_with_kvcache(q, pool, 512, 0.05, cache_seqlens=250, page_table=ids, return_softmax_lse=True)
    rows = pool[ids].reshape(-1, D)[:250]
    compare(q, [rows], [250], 512, 0.05, out, lse, None, range(16), BF)


EXP = [
    # dtype, B, M, N, H, dn, dr, lens, causal
    (BF, 1, 1, 1, 1, 128, 64, [1], True),
    (BF, 1, 300, 300, 2, 128, 64, [300], True),
    (F16, 2, 257, 1000, 3, 128, 64, [1000, 100], True),
    (F32, 2, 77, 130, 3, 64, 32, [130, 20], True),
    (BF, 3, 31, 200, 2, 64, 64, [200, 0, 31], True),
    (F16, 2, 513, 600, 1, 64, 32, [600, 513], True),
    (BF, 2, 100, 333, 2, 128, 32, [333, 64], False),
    (F16, 2, 1, 3000, 4, 128, 64, [3000, 7], False),
    (F32, 2, 40, 100, 2, 128, 64, [100, 0], False),
    (BF, 1, 64, 5000, 2, 128, 64, [5000], True),
]


def make_exp(dtype, B, M, N, H, dn, dr, lens, seed=0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    kv = torch.randn((B, N, H, 2 * dn), generator=g, device="cuda").to(dtype)
    pe = torch.randn((B, N, dr), generator=g, device="cuda").to(dtype)
    q = (torch.randn((B, M, H, dn + dr), generator=g, device="cuda") * 1.5).to(dtype)
    for b, n in enumerate(lens):
        kv[b, n:] = math.nan
        pe[b, n:] = math.nan
    return q, kv[..., :dn], pe, kv[..., dn:], torch.tensor(lens, dtype=torch.int64, device="cuda")


def compare_exp(q, k, pe, v, lens, causal, scale, out, lse, heads, dtype, rows=None):
    M = q.shape[1]
    rows = list(range(M)) if rows is None else rows
    for b, n in enumerate(lens):
        seen = oracle.visible(M, n, causal=causal)
        for h in heads:
            x = np.concatenate([f64(k[b, :n, h]), f64(pe[b, :n])], -1)
            y = f64(v[b, :n, h])
            ref = oracle.attention(f64(q[b, rows, h]), x, y, scale, [seen[m] for m in rows])
            check(out[:, rows], lse[:, :, rows], b, h, ref, q.shape[3], dtype, n, np.abs(y).max() if n else 0.0)


@pytest.mark.parametrize("dtype,B,M,N,H,dn,dr,lens,causal", EXP)
def test_expanded(gpu, dtype, B, M, N, H, dn, dr, lens, causal):
    q, k, pe, v, sl = make_exp(dtype, B, M, N, H, dn, dr, lens, seed=M)
    out, lse = latent_attn_expanded(q, k, pe, v, cache_seqlens=sl, causal=causal, return_softmax_lse=True)
    torch.cuda.synchronize()
    compare_exp(q, k, pe, v, lens, causal, (dn + dr) ** -0.5, out, lse, range(H), dtype)


@pytest.mark.parametrize("dtype", [BF, F16])
def test_expanded_long(gpu, dtype):
    """A prompt of many blocks and tiles, checked at rows on both sides of their borders."""
    M = 2500
    q, k, pe, v, sl = make_exp(dtype, 1, M, M, 2, 128, 64, [M], seed=5)
    out, lse = latent_attn_expanded(q, k, pe, v, cache_seqlens=sl, return_softmax_lse=True)
    rows = sorted({0, 1, 31, 32, 33, 255, 256, 257, 511, 512, 1000, 2047, 2048, 2303, 2304, 2498, 2499})
    compare_exp(q, k, pe, v, [M], True, 192 ** -0.5, out, lse, range(2), dtype, rows)


@pytest.mark.parametrize("dtype", [BF, F16, F32])
def test_expanded_hidden_values_and_growing_scores(gpu, dtype):
    M, n = 300, 340
    q, k, pe, v, sl = make_exp(dtype, 1, M, n, 2, 64, 64, [n], seed=6)
    v[0, n - 2, 1, 5] = math.inf
    v[0, n - 30, 0, 0] = math.nan
    out, lse = latent_attn_expanded(q, k, pe, v, return_softmax_lse=True)
    seen = oracle.visible(M, n)
    for h, hit in ((1, n - 2), (0, n - 30)):
        rows = [m for m in range(M) if hit not in seen[m]]
        y = f64(v[0, :, h])
        y[hit] = 0
        x = np.concatenate([f64(k[0, :, h]), f64(pe[0])], -1)
        ref = oracle.attention(f64(q[0, rows, h]), x, y, 128 ** -0.5, [seen[m] for m in rows])
        check(out[:, rows], lse[:, :, rows], 0, h, ref, 128, dtype, n, np.abs(y).max())
        assert not torch.isfinite(out[0, [m for m in range(M) if hit in seen[m]], h].float()).all(-1).any()
    # Scores that grow by far more than a tile's bound from tile to tile.
    k = torch.zeros((1, n, 1, 64), dtype=dtype, device=gpu)
    k[0, :, 0, 0] = (torch.arange(n, device=gpu) // 8).to(dtype)
    q = torch.zeros((1, 40, 1, 96), dtype=dtype, device=gpu)
    q[..., 0] = 64.0
    pe = torch.zeros((1, n, 32), dtype=dtype, device=gpu)
    v = torch.randn((1, n, 1, 64), device=gpu).to(dtype)
    out, lse = latent_attn_expanded(q, k, pe, v, softmax_scale=1.0, return_softmax_lse=True)
    compare_exp(q, k, pe, v, [n], True, 1.0, out, lse, [0], dtype)


def test_streams_graphs_and_repeats(gpu):
    """Captured and replayed calls, calls on two streams at once, and bit-equal repeats."""
    lens = [1500, 0, 777]
    q, kv, table, sl, _, rows = make(BF, 3, 1, 32, 512, 64, 16, lens, False, seed=4)
    qe, k, pe, v, sle = make_exp(BF, 2, 300, 700, 4, 128, 64, [700, 300], seed=4)

    def both():
        return (*latent_attn_with_kvcache(q, kv, 512, 0.05, cache_seqlens=sl, page_table=table, return_softmax_lse=True),
                *latent_attn_expanded(qe, k, pe, v, cache_seqlens=sle, return_softmax_lse=True))

    want = both()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = both()
    for i in range(4):
        if i == 2:
            sl[1] = 0  # (the same value again: eager work between the replays)
        for t in got:
            t.fill_(7)
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(want, got):
            assert torch.equal(a, b), i
        other = both()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(want, other))
    s1, s2 = torch.cuda.Stream(device=gpu), torch.cuda.Stream(device=gpu)
    with torch.cuda.stream(s1):
        r1 = both()
    with torch.cuda.stream(s2):
        r2 = both()
    torch.cuda.synchronize()
    for a, b, c in zip(want, r1, r2):
        assert torch.equal(a, b) and torch.equal(a, c)


def test_outputs_beside_the_rows_stay(gpu):
    """Rows of a larger output that the call does not own are left as they were."""
    from diffspec_mi355x import _ext
    q, kv, table, sl, _, rows = make(BF, 2, 3, 5, 512, 64, 16, [100, 2], False, seed=8)
    big = torch.full((2, 4, 7, 520), 3.0, dtype=BF, device=gpu)
    out = big[:, :3, 1:6, 4:516]
    lib = _ext.load()
    n = 7 * 16
    nws = lib.dsv_latent_workspace_bytes(2, 3, 5, 512, _ext.DSV_BF16, n, 0, 0)
    ws, ptr = _ext.scratch(nws, gpu)
    _ext.check(lib.dsv_latent_attention(_ext.desc(q), _ext.desc(kv), 512, _ext.desc(table), _ext.desc(sl), n, 0.05, _ext.desc(None),
                                        _ext.desc(out), _ext.desc(None), ptr, nws, _ext.stream_of(gpu)), "latent attention")
    compare(q, rows, [100, 2], 512, 0.05, out, None, None, range(5), BF)
    big[:, :3, 1:6, 4:516] = 3.0
    assert (big == 3.0).all()


@pytest.mark.parametrize("dtype", [BF, F16, F32])
@pytest.mark.parametrize("od", [BF, F16, F32])
def test_expanded_into_strided_outputs(gpu, dtype, od):
    """Rows at any stride, joined from partials (one head of many keys) and whole; what lies between them stays."""
    from diffspec_mi355x import _ext
    lib = _ext.load()
    for M, N, H in ((5, 4000, 1), (40, 50, 3)):
        q, k, pe, v, sl = make_exp(dtype, 2, M, N, H, 64, 32, [N, M], seed=M)
        big = torch.full((2, M + 1, H + 2, 67), 3.0, dtype=od, device=gpu)
        out = big[:, :M, 1:1 + H, 1:65]
        lse = torch.full((2, M, H, 2), 5.0, device=gpu)[..., 0].transpose(1, 2)
        nws = lib.dsv_latent_workspace_bytes(2, M, H, 64, _ext.desc(q).dtype, N, 0, 1)
        ws, ptr = _ext.scratch(nws, gpu)
        _ext.check(lib.dsv_latent_expanded(_ext.desc(q), _ext.desc(k), _ext.desc(pe), _ext.desc(v), _ext.desc(sl), N, 1, 0.1,
                                           _ext.desc(out), _ext.desc(lse), ptr, nws, _ext.stream_of(gpu)), "expanded")
        compare_exp(q, k, pe, v, [N, M], True, 0.1, out, lse, range(H), dtype)
        out.fill_(3.0)
        assert (big == 3.0).all()


@pytest.mark.parametrize("dtype", [BF, F16, F32])
def test_expanded_shared_and_strided_inputs(gpu, dtype):
    """Keys and values shared by the heads or the sequences (stride 0), heads before tokens, one length for all."""
    B, M, N, H, dn, dr = 2, 33, 290, 3, 128, 32
    g = torch.Generator(device="cuda").manual_seed(11)
    rnd = lambda *s: torch.randn(s, generator=g, device=gpu).to(dtype)  # noqa: E731
    q = rnd(B, H, M, dn + dr).transpose(1, 2)
    k = rnd(1, H, N, dn).transpose(1, 2).expand(B, N, H, dn)
    v = rnd(B, N, 1, dn).expand(B, N, H, dn)
    pe = rnd(1, N, dr + 8)[..., :dr].expand(B, N, dr)
    for n, causal in ((N, True), (64, False), (torch.tensor(270, device=gpu), True)):
        out, lse = latent_attn_expanded(q, k, pe, v, cache_seqlens=n, causal=causal, return_softmax_lse=True)
        compare_exp(q, k, pe, v, [int(n)] * B, causal, (dn + dr) ** -0.5, out, lse, range(H), dtype)
    one = rnd(B, 1, H, dn).expand(B, N, H, dn)  # (all keys alike: the mean of the values)
    out, lse = latent_attn_expanded(q, one, pe[:, :1].expand(B, N, dr), v, causal=False, return_softmax_lse=True)
    compare_exp(q, one, pe[:, :1].expand(B, N, dr), v, [N] * B, False, (dn + dr) ** -0.5, out, lse, range(H), dtype)


@pytest.mark.parametrize("dtype", [BF, F16])
def test_expanded_units_of_their_own(gpu, dtype):
    """So many heads and row blocks that no sequence's keys are shared out."""
    M, H = 2100, 115
    q, k, pe, v, sl = make_exp(dtype, 2, M, M, H, 64, 32, [M, 1500], seed=12)
    out, lse = latent_attn_expanded(q, k, pe, v, cache_seqlens=sl, return_softmax_lse=True)
    rows = [0, 599, 600, 601, 1023, 1024, 2047, 2099]
    compare_exp(q, k, pe, v, [M, 1500], True, 96 ** -0.5, out, lse, [0, 57, 114], dtype, rows)


@pytest.mark.parametrize("dtype", [BF, F16])
@pytest.mark.parametrize("M,N", [(1, 6000), (300, 700)])
def test_expanded_very_large_scores(gpu, dtype, M, N):
    """Scores beyond 2^21, whose product with the scale a fused exponent would round away, growing along the keys
    (in partials, too).  Scores are single products of short numbers, exact in fp32, so the weights are those of
    exact differences; the bounds are those of the file's head with delta 0, the product of a difference of up to
    40 with the scale (2^-23 of it) in its place."""
    k = torch.zeros((1, N, 1, 64), dtype=dtype, device=gpu)
    k[0, :, 0, 0] = (1024 + torch.arange(N, device=gpu) // 64).to(dtype)
    k[0, :, 0, 1] = (torch.arange(N, device=gpu) % 7).to(dtype)
    q = torch.zeros((1, M, 1, 96), dtype=dtype, device=gpu)
    q[..., 0] = 4096.0
    q[..., 1] = 1.0
    pe = torch.zeros((1, N, 32), dtype=dtype, device=gpu)
    v = torch.randn((1, N, 1, 64), device=gpu).to(dtype)
    out, lse = latent_attn_expanded(q, k, pe, v, softmax_scale=1.0, return_softmax_lse=True)
    x, y = f64(k[0, :, 0]), f64(v[0, :, 0])
    s = 4096 * x[:, 0] + x[:, 1]
    assert s.max() > 2 ** 22 and np.array_equal(np.float32(s), s)
    u = torch.finfo(dtype).eps / 2
    for m in sorted({0, M // 2, M - 1}):
        n = N - M + m + 1
        w = np.exp(s[:n] - s[:n].max())
        ref, mass = (w @ y[:n]) / w.sum(), (w @ np.abs(y[:n])) / w.sum()
        tol = mass * (u + 80 * 2.0 ** -24 + (n + 64) * 2.0 ** -24 + 2.0 ** -22) * 1.01 + u * np.abs(ref) + n * 2.0 ** -34 * np.abs(y).max()
        assert (np.abs(f64(out[0, m, 0]) - ref) <= tol).all(), m
        want = s[:n].max() + math.log(w.sum())
        assert abs(float(lse[0, 0, m]) - want) <= 2.0 ** -21 * want


@pytest.mark.parametrize("dtype", [BF, F32])
def test_absorbed_odd_lengths_and_pages(gpu, dtype):
    """Lengths below 0 and beyond 32 bits, sequences that share pages, numbers outside the pool (clamped to it)."""
    q, kv, _, _, _, rows = make(dtype, 1, 2, 4, 256, 32, 16, [96], False, seed=13, spare=0)
    q = q.expand(4, 2, 4, 288)
    kv = torch.randn((6, 16, 288), device=gpu).to(dtype)
    table = torch.tensor([[0, 1, 2, 3], [3, 1, 0, 5], [-7, 2, 99, 5], [1, 1, 1, 1]], device=gpu)
    lens = torch.tensor([-5, (1 << 40) + 3, 64, 33], device=gpu)
    out, lse = latent_attn_with_kvcache(q, kv, 256, 0.06, cache_seqlens=lens, page_table=table, return_softmax_lse=True)
    n = [0, 64, 64, 33]
    seq = [kv[table[b].clamp(0, 5)].reshape(64, 288)[:n[b]] for b in range(4)]
    compare(q, seq, n, 256, 0.06, out, lse, None, range(4), dtype)
    low = lens.clamp(-5, 200).int()
    again = latent_attn_with_kvcache(q, kv, 256, 0.06, cache_seqlens=low, page_table=table.int())
    assert torch.equal(out, again)


def test_two_graphs_and_new_lengths(gpu):
    """Two captured graphs replayed in turn while their lengths, tables and caches change."""
    lens = [4000, 90, 1500]
    q, kv, table, sl, _, rows = make(BF, 3, 1, 64, 512, 64, 16, lens, False, seed=14)
    kv.nan_to_num_(0.5)
    table.clamp_(min=0)
    calls = [lambda: latent_attn_with_kvcache(q, kv, 512, 0.05, cache_seqlens=sl, page_table=table, return_softmax_lse=True),
             lambda: latent_attn_with_kvcache(q[:, :, :16], kv, 512, 0.05, cache_seqlens=sl, page_table=table, return_softmax_lse=True)]
    graphs, outs = [], []
    for call in calls:
        call()
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(call())
        graphs.append(g)
    for i in range(4):
        sl.copy_(torch.tensor([[4000, 90, 1500], [1, 4000, 0], [64, 65, 63], [4000, 4000, 4000]][i], device=gpu))
        table.copy_(table[torch.tensor([1, 2, 0], device=gpu)])
        kv[i].fill_(0.25)
        for g in graphs:
            g.replay()
        for got, call in zip(outs, calls):
            want = call()
            torch.cuda.synchronize()
            assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1]), i


@pytest.mark.parametrize("dtype", [BF, F16, F32])
def test_absorbed_whole_range_of_batches(gpu, dtype):
    """Many short sequences of random lengths (each CU's share holds several), and rows left empty."""
    rng = np.random.default_rng(15)
    B = 600
    lens = [int(x) for x in rng.integers(0, 150, B)]
    q, kv, table, sl, _, rows = make(dtype, B, 2, 3, 256, 64, 16, lens, False, seed=15)
    out, lse = latent_attn_with_kvcache(q, kv, 256, 0.06, cache_seqlens=sl, page_table=table, return_softmax_lse=True)
    pick = sorted({0, 599, *(int(x) for x in rng.integers(0, B, 60)), *(i for i, n in enumerate(lens) if n < 3)})
    for b in pick:
        compare(q[b:b + 1], rows[b:b + 1], lens[b:b + 1], 256, 0.06, out[b:b + 1], lse[b:b + 1], None, range(3), dtype)
    assert torch.isfinite(out.float()).all()


@pytest.mark.parametrize("dtype", [BF, F16, F32])
@pytest.mark.parametrize("lens", [[20000], [900, 0, 15000]])
def test_absorbed_many_partials_a_row(gpu, dtype, lens):
    """Few rows over many keys: more partials a row than a wave joins at once, some without a key of the row."""
    B = len(lens)
    q, kv, table, sl, _, rows = make(dtype, B, 2, 3, 256, 64, 64, lens, False, seed=16)
    out, lse = latent_attn_with_kvcache(q, kv, 256, 0.06, cache_seqlens=sl, page_table=table, return_softmax_lse=True)
    compare(q, rows, lens, 256, 0.06, out, lse, None, range(3), dtype)
    # All weight on a token of the first piece, then of the last: the joined maximum is another piece's.
    for at in (3, lens[-1] - 2):
        one = rows[-1].clone()
        one[at] = (q[-1, 0, 0].float() * 3).to(dtype)
        page = table[-1, at // 64]
        kv[page, at % 64] = one[at]
        out, lse = latent_attn_with_kvcache(q, kv, 256, 0.5, cache_seqlens=sl, page_table=table, return_softmax_lse=True)
        compare(q[-1:], [one], lens[-1:], 256, 0.5, out[-1:], lse[-1:], None, range(3), dtype)
        kv[page, at % 64] = rows[-1][at]


@pytest.mark.parametrize("dtype", [BF, F32])
def test_expanded_many_partials_a_row(gpu, dtype):
    q, k, pe, v, sl = make_exp(dtype, 1, 3, 14000, 2, 128, 64, [14000], seed=17)
    out, lse = latent_attn_expanded(q, k, pe, v, cache_seqlens=sl, return_softmax_lse=True)
    compare_exp(q, k, pe, v, [14000], True, 192 ** -0.5, out, lse, range(2), dtype)
