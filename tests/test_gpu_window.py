"""window_attn_with_kvcache against float64 sums over the visible keys."""

import random

import numpy as np
import pytest
import torch

from diffspec_mi355x import workloads as wl
from diffspec_mi355x.runtime.window_attention import window_attn_with_kvcache
from oracle import window as oracle

pytestmark = pytest.mark.gpu

BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32


def bounds(dtype, out_dtype, want, lse, absum, reach, n, D, vmax):
    """Error bounds of out and lse, from the roundings that the operator makes.

    Scores: D products summed in fp32, off by (D + 4) 2^-24 of the sum of |q k|;
    the exponent's argument and the exponential add 2^-21.  Probabilities
    round to the inputs' 16-bit type: half a step of the value, or, below
    fp16's normal range, 2^-25 of the running maximum's, which the sum holds
    at least once.  Sums over n keys in fp32; the output's own rounding.
    """
    u = 2.0 ** -24
    score = (D + 4) * u * reach.max(initial=0.0) + 2.0 ** -21
    rel = 2 * score + 2 * (n + 16) * u
    half_p = 0.0 if dtype == F32 else torch.finfo(dtype).eps / 2
    tol = absum * (rel + half_p) + np.abs(want) * (torch.finfo(out_dtype).eps / 2) * 1.01 + 1e-30
    if dtype == F16:
        tol = tol + n * 2.0 ** -25 * vmax
    if out_dtype == F16:
        tol = tol + 2.0 ** -25
    return tol, score + (n + 16) * u + 2.0 ** -22 * (1.0 + np.abs(np.where(np.isfinite(lse), lse, 0.0)))


class Case:
    def __init__(self, gpu, B, M, H, Hk, D, lens, dtype, page=0, seed=0, scale=1.0, cap=None, spare=3):
        g = torch.Generator().manual_seed(seed)
        rng = np.random.default_rng(seed)
        self.gpu, self.B, self.M, self.lens, self.dtype, self.page = gpu, B, M, list(lens), dtype, page
        cap = cap or max(max(lens), 1)
        r = lambda *s: torch.randn(s, generator=g).to(dtype)  # noqa: E731
        self.q = (torch.randn((B, M, H, D), generator=g) * scale).to(dtype).to(gpu)
        self.table = None
        if page:
            n_log = -(-cap // page)
            P = B * n_log + spare
            self.table = torch.from_numpy(rng.permutation(P)[:B * n_log].reshape(B, n_log).astype(np.int32)).to(gpu)
            self.k, self.v = r(P, Hk, page, D).to(gpu), r(P, Hk, page, D).to(gpu)
        else:
            self.k, self.v = r(B, cap, Hk, D).to(gpu), r(B, cap, Hk, D).to(gpu)

    def rows(self, b):
        """K and V rows of sequence b in logical order, float64."""
        if self.table is None:
            return self.k[b].double().cpu().numpy(), self.v[b].double().cpu().numpy()
        t = self.table[b].long().clamp(0, self.k.shape[0] - 1)
        f = lambda x: x[t].transpose(1, 2).reshape(-1, x.shape[1], x.shape[3]).double().cpu().numpy()  # noqa: E731
        return f(self.k), f(self.v)

    def slot(self, x, b, n):
        """The row of token n in K or V, a view."""
        return x[b, n] if self.table is None else x[int(self.table[b, n // self.page]), :, n % self.page]

    def check(self, window, sinks, parent=None, lens_arg="tensor", out_dtype=None, result=None):
        od = out_dtype or self.dtype
        lens = torch.tensor(self.lens, dtype=torch.int32, device=self.gpu) if lens_arg == "tensor" else lens_arg
        par = None if parent is None else torch.tensor(parent, dtype=torch.int32, device=self.gpu)
        if result is None:
            result = window_attn_with_kvcache(self.q, self.k, self.v, window, sinks, lens, self.table, par, True, out_dtype)
        out, lse = (x.double().cpu().numpy() for x in result)
        assert result[0].dtype == od and result[1].dtype == F32
        for b in range(self.B):
            p = None if parent is None else (parent[b] if isinstance(parent[0], list) else parent)
            keys = oracle.visible(self.M, self.lens[b], window, sinks, p)
            k, v = self.rows(b)
            want, wl_, absum, reach = oracle.attend(self.q[b].double().cpu().numpy(), k, v, keys)
            seen = np.unique(np.concatenate(keys)) if keys else np.zeros(0, dtype=np.int64)
            vmax = np.abs(v[seen]).max(initial=0.0)
            n = max((x.size for x in keys), default=0)
            tol, ltol = bounds(self.dtype, od, want, wl_, absum, reach, n, k.shape[2], vmax)
            bad = ~(np.abs(out[b] - want) <= tol)
            assert not bad.any(), (b, np.argwhere(bad)[:3], out[b][bad][:3], want[bad][:3], tol[bad][:3])
            empty = ~np.isfinite(wl_)
            assert (lse[b][empty] == -np.inf).all()
            assert (out[b].transpose(1, 0, 2)[empty] == 0).all()
            d = np.abs(np.where(empty, 0.0, lse[b]) - np.where(empty, 0.0, wl_))
            assert (d <= ltol).all(), (b, d.max())
        return result


SIZES = [
    # B, M, H, Hk, D, lens, window, sinks, page
    (1, 1, 1, 1, 64, [1], 1, 0, 0),
    (1, 1, 8, 2, 128, [300], 40, 4, 16),
    (3, 1, 8, 1, 128, [0, 1, 500], 100, 3, 0),
    (2, 1, 14, 2, 64, [777, 31], 65, 33, 8),
    (2, 1, 32, 1, 128, [90, 64], 7, 0, 4),
    (2, 5, 4, 4, 128, [3, 64], 16, 2, 1),
    (2, 7, 6, 2, 64, [200, 4], 1, 5, 2),
    (3, 33, 8, 8, 128, [33, 32, 700], 50, 64, 0),
    (1, 64, 8, 2, 128, [64], 1000, 0, 16),
    (1, 100, 5, 1, 64, [1000], 96, 70, 64),
    (2, 130, 4, 2, 128, [131, 900], 33, 1, 128),
    (1, 300, 12, 4, 64, [300], 128, 0, 0),
    (1, 257, 8, 2, 128, [1500], 512, 130, 32),
]


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("case", SIZES, ids=lambda c: "-".join(map(str, c[:5])))
def test_causal(gpu, case, dtype):
    B, M, H, Hk, D, lens, window, sinks, page = case
    Case(gpu, B, M, H, Hk, D, lens, dtype, page, seed=M + H).check(window, sinks)


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("M,H,Hk,D,lens,window,sinks,page", [
    (1, 4, 2, 64, [50, 1], 9, 2, 16), (9, 8, 2, 128, [9, 300], 40, 4, 0), (16, 32, 8, 128, [700, 33], 5, 30, 16),
    (64, 8, 2, 128, [64, 1000], 200, 16, 32), (65, 4, 4, 64, [500, 40], 3, 470, 0), (130, 8, 1, 128, [400, 131], 64, 140, 1),
    (200, 4, 1, 64, [205, 900], 600, 0, 64)])
def test_tree(gpu, M, H, Hk, D, lens, window, sinks, page, dtype):
    """Trees by batch, windows shorter than the trees' depth, sinks that reach into the tree, len < M."""
    parents = [wl.make_tree(M, max_depth=max(8, M), max_outdeg=3, seed=M + i)[0] for i in range(2)]
    c = Case(gpu, 2, M, H, Hk, D, lens, dtype, page, seed=M)
    c.check(window, sinks, parents)
    c.check(window, sinks, parents[0])


def test_tree_shapes(gpu):
    """Chains, stars, forests, cycles and parents out of range; 1024 nodes."""
    c = Case(gpu, 1, 70, 4, 2, 64, [170], BF16, 16, seed=1)
    for parent in [list(range(-1, 69)), [-1] + [0] * 69, [-1] * 70, [i if i % 9 == 0 else i - 1 for i in range(70)],
                   [69] + list(range(69)), [100 if i % 5 == 0 else i - 1 for i in range(70)]]:
        c.check(20, 4, parent)
    M = 1024
    Case(gpu, 1, M, 1, 1, 64, [M + 40], BF16, 0, seed=2).check(100, 3, wl.make_tree(M, max_depth=40, max_outdeg=4, seed=3)[0])
    # A chain is causal.
    c = Case(gpu, 2, 48, 8, 2, 128, [48, 300], F16, 16, seed=4)
    a = c.check(30, 2, list(range(-1, 47)))
    b = c.check(30, 2)
    assert torch.allclose(a[0].float(), b[0].float(), atol=2e-3, rtol=0)


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("M,H", [(70, 4), (12, 2)])
def test_cyclic_tree_in_a_long_window(gpu, M, H, dtype):
    """Nodes whose parents form one cycle: a walk ends after M nodes, at depth M - 1 (every prefix border shows it)."""
    cycle = [M - 1] + list(range(M - 1))
    c = Case(gpu, 1, M, H, 2, 64, [M + 100], dtype, 16, seed=M)
    for window, sinks in [(100, 0), (M + 1, 3), (M - 1, 0), (30, M + 100 - 5), (1, 100 + M - 1), (1, 100 + M)]:
        c.check(window, sinks, cycle)


@pytest.mark.parametrize("dtype", [BF16, F32])
def test_lengths(gpu, dtype):
    """Lengths as an int, a 0-d and an int64 tensor, None; beyond the cache; a window beyond every length."""
    c = Case(gpu, 2, 3, 4, 2, 64, [100, 100], dtype, 16, cap=112)
    want = c.check(1 << 40, 1 << 45, lens_arg=100)
    for arg in [torch.tensor(100), torch.tensor([100, 100])]:
        got = c.check(1 << 40, 1 << 45, lens_arg=arg.to(gpu))
        assert torch.equal(want[0], got[0]) and torch.equal(want[1], got[1])
    c.lens = [112, 112]
    c.check(20, 3, lens_arg=None)
    c.check(20, 3, lens_arg=torch.tensor([500, 112], device=gpu))
    c.lens = [0, 2]
    c.check(20, 3, lens_arg=torch.tensor([-5, 2], device=gpu))
    c.lens = [0, 0]
    c.check(20, 3, lens_arg=0)


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("page,M", [(0, 1), (16, 1), (0, 20), (16, 20), (8, 90), (0, 300)])
def test_hidden_values(gpu, page, M, dtype):
    """NaN and infinities wherever a row sees nothing never reach it; missing pages are not read as keys."""
    lens, window, sinks = [400, 3 * M + 50], 60, 5
    cap = max(lens) + 40
    c = Case(gpu, 2, M, 8, 2, 64, lens, dtype, page, cap=cap, seed=M)
    hidden = []
    for b in range(2):
        keys = oracle.visible(M, lens[b], window, sinks)
        seen = set(np.concatenate(keys).tolist())
        hidden.append([n for n in range(cap) if n not in seen])
        for i, n in enumerate(hidden[b]):
            c.slot(c.k, b, n)[:] = [float("nan"), float("inf"), -float("inf")][i % 3]
            c.slot(c.v, b, n)[:] = [float("inf"), float("nan"), -float("inf")][i % 3]
    if page:
        for b in range(2):
            for j in range(c.table.shape[1]):
                if all(n in hidden[b] for n in range(j * page, (j + 1) * page)):
                    c.table[b, j] = [-1, -2 ** 31, 2 ** 31 - 1][j % 3]
    c.check(window, sinks)


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("M,G", [(8, 4), (40, 1), (200, 2)])
def test_values_hidden_from_some_rows(gpu, M, G, dtype):
    """A V entry that is infinite or NaN reaches the rows that see its key, and no others."""
    n, window, sinks = M + 100, 30, 2
    c = Case(gpu, 1, M, 2 * G, 2, 64, [n], dtype, 0, seed=3)
    keys = oracle.visible(M, n, window, sinks)
    for key in (n - M - window + 3, n - M // 2, n - 1):
        for kind in (float("inf"), float("nan")):
            good = c.v.clone()
            c.v[0, key, 1, 5] = kind
            out = window_attn_with_kvcache(c.q, c.k, c.v, window, sinks).cpu()
            c.v.copy_(good)
            ref = window_attn_with_kvcache(c.q, c.k, c.v, window, sinks).cpu()
            for m in range(M):
                sees = key in keys[m]
                assert torch.isfinite(out[0, m, G:, 5]).all() == (not sees), (m, key, kind)
                if not sees:
                    # (The other keys' sums, of the same values.)
                    assert torch.allclose(out[0, m].float(), ref[0, m].float(), rtol=2 ** -6, atol=2 ** -6)
            assert torch.equal(out[0, :, :G], ref[0, :, :G])


def test_masks_of_scores(gpu):
    """Very large, very small and infinite scores."""
    for dtype in (BF16, F16, F32):
        c = Case(gpu, 1, 6, 4, 2, 64, [90], dtype, 0, seed=8, scale=30.0)
        c.check(40, 4)
        c = Case(gpu, 1, 6, 4, 2, 64, [90], dtype, 0, seed=9, scale=0.0)
        c.check(40, 4)
    c = Case(gpu, 1, 40, 4, 2, 64, [90], BF16, 0, seed=8)
    c.k[0, 85] = float("nan")   # seen by the last rows only
    out, lse = window_attn_with_kvcache(c.q, c.k, c.v, 4, 0, return_softmax_lse=True)
    sees = torch.tensor([85 in x for x in oracle.visible(40, 90, 4, 0)], device=gpu)
    assert torch.equal(torch.isnan(out[0]).all(-1).all(-1), sees)
    assert torch.equal(torch.isnan(lse[0]).all(0), sees)


@pytest.mark.parametrize("M", [5, 70])
def test_strides_and_output_types(gpu, M):
    """Heads before tokens, padded rows, shared tables, an int64 table, every output type."""
    c = Case(gpu, 2, M, 6, 2, 64, [120, 77], BF16, 16, seed=5)
    want = c.check(50, 3)
    big = torch.zeros(2, 6, M + 2, 80, dtype=BF16, device=gpu)
    qv = big[:, :, 1:M + 1, :64].transpose(1, 2)
    qv.copy_(c.q)
    pool = torch.zeros(2, c.k.shape[0], 16, 2, 72, dtype=BF16, device=gpu)
    kv, vv = (pool[i, ..., :64].transpose(1, 2) for i in range(2))
    kv.copy_(c.k), vv.copy_(c.v)
    table = torch.full((2, 20), -1, dtype=torch.int64, device=gpu)
    table[:, :c.table.shape[1]] = c.table
    lens = torch.tensor([120, 77], device=gpu)
    got = window_attn_with_kvcache(qv, kv, vv, 50, 3, lens, table[:, :c.table.shape[1]], None, True)
    assert torch.equal(want[0], got[0]) and torch.equal(want[1], got[1])
    for od in (BF16, F16, F32):
        c.check(50, 3, out_dtype=od)
    c.table = c.table[:1].expand(2, -1).contiguous()
    got = window_attn_with_kvcache(c.q, c.k, c.v, 50, 3, lens, c.table[0], None, True)
    c.check(50, 3, result=got)


@pytest.mark.parametrize("M", [5, 70])
def test_c_abi_strided_outputs(gpu, dsv_lib, M):
    """Outputs at strides of their own: rows between theirs stay as they were."""
    from diffspec_mi355x import _ext
    for dtype in (BF16, F32):
        c = Case(gpu, 2, M, 6, 2, 64, [120, 3], dtype, 0, seed=6)
        for pad in (1, 8):
            big = torch.full((2, M + 1, 6, 64 + pad), 7.0, dtype=dtype, device=gpu)
            out = big[:, 1:, :, :64]
            lbig = torch.full((2, M, 7), 7.0, device=gpu)
            lse = lbig[:, :, :6].transpose(1, 2)
            d = _ext.desc
            lens = torch.tensor(c.lens, device=gpu)
            n = dsv_lib.dsv_window_workspace_bytes(2, M, 6, 2, 64, d(c.q).dtype, 120, 50, 3, 0)
            ws = _ext.workspace(n, gpu)
            rc = dsv_lib.dsv_window_attention(d(c.q), d(c.k), d(c.v), d(None), d(lens), -1, 50, 3, d(None), d(out), d(lse),
                                              ws.data_ptr(), n, _ext.stream_of(gpu))
            assert rc == 0, _ext.last_error()
            c.check(50, 3, result=(out, lse))
            assert bool((big[:, 0] == 7).all()) and bool((big[..., 64:] == 7).all()) and bool((lbig[:, :, 6:] == 7).all())


@pytest.mark.parametrize("M", [4, 40])
def test_long_cache_beyond_32_bits(gpu, M):
    """Offsets past 2^32 bytes into the cache, dense and paged."""
    N = 1 << 20
    k = torch.zeros(1, N, 16, 128, dtype=BF16, device=gpu)   # 4 GiB a half
    v = torch.zeros_like(k)
    c, window = Case(gpu, 1, M, 32, 16, 128, [64], BF16, 0, seed=7), 62 - M
    k[:, N - 61:N], v[:, N - 61:N] = c.k[:, 3:], c.v[:, 3:]
    k[:, :3], v[:, :3] = c.k[:, :3], c.v[:, :3]
    # The last 61 keys and 3 sinks are the small cache's 64 keys.
    a = window_attn_with_kvcache(c.q, k, v, window, 3, return_softmax_lse=True)
    small = window_attn_with_kvcache(c.q, c.k, c.v, window, 3, return_softmax_lse=True)
    assert torch.allclose(a[0].float(), small[0].float(), rtol=2 ** -7, atol=2 ** -7)
    assert torch.allclose(a[1], small[1], rtol=1e-5, atol=1e-5)
    pages = lambda x: x.view(N // 64, 64, 16, 128).transpose(1, 2)  # noqa: E731
    b = window_attn_with_kvcache(c.q, pages(k), pages(v), window, 3, None, torch.arange(N // 64, device=gpu), None, True)
    assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])


def test_random(gpu):
    rng = random.Random(11)
    for i in range(60):
        Hk = rng.choice([1, 2, 3])
        M = rng.choice([1, 1, 2, 3, 17, 40, 75, 129])
        B = rng.choice([1, 2, 3])
        hi = rng.choice([20, 100, 700])
        lens = [rng.randint(0, hi) for _ in range(B)]
        tree = rng.random() < 0.4
        c = Case(gpu, B, M, Hk * rng.choice([1, 2, 5, 8]), Hk, rng.choice([64, 128]), lens, rng.choice([BF16, F16, F32]),
                 rng.choice([0, 1, 4, 16, 64]), seed=i, cap=hi + rng.randint(0, 40))
        parent = wl.make_tree(M, max_depth=max(6, M), max_outdeg=4, seed=i)[0] if tree else None
        print(i, B, M, lens, tree, flush=True)
        c.check(rng.choice([1, 2, 15, 33, 64, 300, 5000]), rng.choice([0, 1, 4, 31, 32, 200]), parent)


def test_streams_and_graphs(gpu):
    """A side stream; two graphs captured with their own workspaces, replayed in turn with other inputs."""
    cs = [Case(gpu, 2, 1, 8, 2, 128, [900, 300], BF16, 16, seed=s) for s in (1, 2)]
    parent = wl.make_tree(12, max_depth=6, max_outdeg=3, seed=1)[0]
    ct = Case(gpu, 1, 12, 8, 2, 128, [500], BF16, 16, seed=3)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    lens = torch.tensor([900, 300], device=gpu)
    par = torch.tensor(parent, device=gpu)
    f = lambda c: window_attn_with_kvcache(c.q, c.k, c.v, 300, 4, lens, c.table, None, True)  # noqa: E731
    ft = lambda: window_attn_with_kvcache(ct.q, ct.k, ct.v, 300, 4, 500, ct.table, par, True)  # noqa: E731
    with torch.cuda.stream(s):
        side = f(cs[0])
    torch.cuda.synchronize()
    want = [f(cs[0]), f(cs[1]), ft()]
    assert torch.equal(side[0], want[0][0])
    graphs, outs = [], []
    for g in (lambda: f(cs[0]), ft):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs.append(g())
        graphs.append(graph)
    for i in range(4):
        cs[0].q.copy_(cs[1].q if i % 2 else cs[0].q)
        eager = f(cs[0])
        for graph in graphs:
            graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(outs[0][0], eager[0]) and torch.equal(outs[0][1], eager[1])
        assert torch.equal(outs[1][0], want[2][0]) and torch.equal(outs[1][1], want[2][1])


@pytest.mark.parametrize("M,page,D", [(20, 16, 64), (20, 8, 128), (3, 64, 128)])
def test_many_tiles_of_one_split(gpu, M, page, D):
    """A workgroup per CU, each over about 90 tiles: paged as dense bit by bit, some heads against float64."""
    lens, window, sinks = [3001, 2950, 64, 2999, 3000, 0, 1500, 2960], 2900, 40
    c = Case(gpu, 8, M, 32, 32, D, lens, BF16, page, seed=M + D)
    lens_t = torch.tensor(lens, device=gpu)
    dense = [x[c.table.long()].transpose(2, 3).reshape(8, -1, 32, D) for x in (c.k, c.v)]
    a = window_attn_with_kvcache(c.q, c.k, c.v, window, sinks, lens_t, c.table, None, True)
    b = window_attn_with_kvcache(c.q, *dense, window, sinks, lens_t, None, None, True)
    assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])
    for i, h in ((0, 5), (3, 31), (6, 0)):
        keys = oracle.visible(M, lens[i], window, sinks)
        k, v = (x[i, :, h:h + 1].double().cpu().numpy() for x in dense)
        want, wl_, absum, reach = oracle.attend(c.q[i, :, h:h + 1].double().cpu().numpy(), k, v, keys)
        tol, ltol = bounds(BF16, BF16, want, wl_, absum, reach, window + sinks, D, np.abs(v).max())
        assert (np.abs(a[0][i, :, h:h + 1].double().cpu().numpy() - want) <= tol).all()
        assert (np.abs(a[1][i, h:h + 1].double().cpu().numpy() - wl_) <= ltol).all()
