"""Slot maps and the latent append, and a decoding step of the latent operators together."""

import math

import numpy as np
import pytest
import torch

from diffspec_mi355x.core.kv_cache import compact_pages, extend_pages, fork_pages, token_slots
from diffspec_mi355x.runtime.cache_state import append_latent_kv
from diffspec_mi355x.runtime.latent_attention import latent_attn_expanded, latent_attn_with_kvcache
from oracle import latent as oracle

pytestmark = pytest.mark.gpu

BF, F16, F32 = torch.bfloat16, torch.float16, torch.float32
KEYS = ("slots", "positions", "requests", "cu_seqlens", "block_table", "lens")


def f64(t):
    return t.detach().double().cpu().numpy()


def check_slots(table, lens, news, page, cap, seqs=None, **kw):
    got = token_slots(table, lens, news, page, cap, seqs=seqs)
    want = oracle.token_slots(table.tolist(), lens.tolist(), news.tolist(), page, cap, None if seqs is None else seqs.tolist())
    for key, w in zip(KEYS, want):
        g = got[key]
        assert g.dtype == (torch.int64 if key == "slots" else torch.int32)
        assert torch.equal(g.cpu().long().reshape(-1), torch.tensor(w, dtype=torch.int64).reshape(-1)), key
    return got


@pytest.mark.parametrize("B,n,page,hi,new,cap", [
    (1, 1, 16, 5, 1, 1), (1, 1, 1, 40, 40, 64), (7, 7, 16, 100, 9, 0), (7, 5, 4, 300, 50, 97), (64, 48, 64, 5000, 1, 64),
    (300, 256, 16, 400, 30, 6000), (2048, 2048, 8, 60, 3, 5000), (2500, 2049, 8, 60, 3, 3000), (2500, 2500, 16, 30, 5, 20000)])
@pytest.mark.parametrize("i64", [False, True])
def test_token_slots(gpu, B, n, page, hi, new, cap, i64):
    rng = np.random.default_rng(B + n)
    dt = torch.int64 if i64 else torch.int32
    n_log = -(-hi // page) + 1
    table = torch.from_numpy(rng.integers(0, 1 << 20, (B, n_log)).astype(np.int32))
    table[rng.random((B, n_log)) < 0.05] = -1
    lens = torch.from_numpy(rng.integers(0, hi + 1, B)).to(dt)
    news = torch.from_numpy(rng.integers(0, new + 1, n)).to(dt)
    seqs = torch.from_numpy(rng.permutation(B)[:n].copy()).to(dt)
    for s in ([seqs, None] if n == B else [seqs]):
        check_slots(table.cuda(), lens.cuda(), news.cuda(), page, cap, None if s is None else s.cuda())


def test_token_slots_odd_requests(gpu):
    """Lengths and counts out of range, sequences out of range or named twice, strided lists, no requests, huge totals."""
    i32 = lambda *x: torch.tensor(x, dtype=torch.int32, device=gpu)  # noqa: E731
    table = torch.arange(12, dtype=torch.int32, device=gpu).view(3, 4)
    check_slots(table, i32(5, 99, -3), i32(7, 20, 1), 4, 40)
    check_slots(table, i32(5, 16, 9), i32(2, -5, 3, 4, 1, 1), 4, 12, i32(1, 1, 1, 2, -1, 3))
    check_slots(table, i32(5, 16, 9), i32(2, 0, 5, 0, 3, 0)[::2], 4, 12, i32(0, 9, 2, 9, 1, 9)[::2])
    check_slots(table[:, :3], i32(12, 12, 12), i32(3, 3, 3), 4, 12)
    check_slots(table, i32(5, 16, 9), i32(), 4, 3, i32())
    wide = torch.zeros((3, 1 << 14), dtype=torch.int32, device=gpu)
    big = 1 << 30
    got = token_slots(wide, i32(big, big, big), i32(big, big, big), 1 << 16, 5)
    assert got["cu_seqlens"].tolist() == [0, big, 2 ** 31 - 1, 2 ** 31 - 1]
    assert got["positions"].tolist() == list(range(5)) and got["slots"].tolist() == list(range(5))


def test_token_slots_captured(gpu):
    table = torch.arange(4000, dtype=torch.int32, device=gpu).view(40, 100)
    lens = torch.full((40,), 300, dtype=torch.int32, device=gpu)
    news = torch.ones(40, dtype=torch.int32, device=gpu)
    token_slots(table, lens, news, 16, 64)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = token_slots(table, lens, news, 16, 64)
    for i in range(3):
        lens += i
        news.fill_(1 + i % 2)
        graph.replay()
        torch.cuda.synchronize()
        want = token_slots(table, lens, news, 16, 64)
        for key in KEYS:
            assert torch.equal(got[key], want[key]), (i, key)


def tables(n_pos, dr, interleaved, dtype=F32):
    ang = torch.arange(n_pos, dtype=torch.float64)[:, None] * 100.0 ** (-torch.arange(0, dr, 2, dtype=torch.float64) / dr)
    ang = ang.repeat_interleave(2, -1) if interleaved else torch.cat([ang, ang], -1)
    return ang.cos().to(dtype).cuda(), ang.sin().to(dtype).cuda()


@pytest.mark.parametrize("dtype", [BF, F16, F32])
@pytest.mark.parametrize("T,dc,dr,H,page,inter,norm,tab", [
    (1, 512, 64, 16, 64, True, True, F32), (5, 256, 32, 0, 16, False, True, None), (130, 512, 64, 3, 8, False, False, F32),
    (67, 8, 16, 2, 1, True, True, F32), (33, 1048, 112, 5, 4, False, True, F32), (9, 2048, 2048, 1, 2, True, True, F32),
    (77, 512, 64, 128, 32, True, True, "same")])
def test_append(gpu, dtype, T, dc, dr, H, page, inter, norm, tab):
    """Bounds: the norm's factor is off by (dc / 2 + 4) 2^-24 (half of the sum of squares' error, root, quotient) and
    two products, a rotation by three roundings of |x cos| + |partner sin|; then half a step of the type."""
    rng = np.random.default_rng(T)
    g = torch.Generator(device="cuda").manual_seed(T)
    kv = torch.randn((T, dc + dr + 16), generator=g, device=gpu).to(dtype)  # (rows with room behind them)
    c, pe = kv[:, :dc], kv[:, dc:dc + dr]
    P = -(-T // page) + 2
    cache = torch.full((P, page, dc + dr), 9.0, dtype=dtype, device=gpu)
    slots = torch.from_numpy(rng.permutation(P * page)[:T].copy())
    slots[rng.random(T) < 0.2] = -1
    if T > 4:
        slots[3] = P * page  # out of range: not stored
    w = torch.randn(dc, generator=g, device=gpu).to(dtype) if norm else None
    cos = sin = pos = None
    if tab is not None:
        cos, sin = tables(50, dr, inter, F32 if tab is F32 else dtype)
        pos = torch.from_numpy(rng.integers(-3, 60, T))
    q = torch.randn((T, H, dr + 8), generator=g, device=gpu).to(dtype)[..., 8:] if H else None
    got = append_latent_kv(c, pe, cache, slots.to(gpu), norm_weight=w, eps=1e-5, cos=cos, sin=sin,
                           positions=None if pos is None else pos.to(torch.int32).to(gpu), interleaved=inter, q_pe=q)
    torch.cuda.synchronize()
    p = None if pos is None else pos.clamp(0, 49).numpy()
    cs, sn = (None, None) if cos is None else (f64(cos)[p], f64(sin)[p])
    want = np.full((P * page, dc + dr), 9.0)
    tol = np.zeros_like(want)
    x, y = f64(c), f64(pe)
    rows = oracle.latent_rows(x, y, None if w is None else f64(w), 1e-5, cs, sn, inter)
    u = torch.finfo(dtype).eps / 2
    err = np.abs(rows) * u * 1.01
    if norm:
        err[:, :dc] += np.abs(rows[:, :dc]) * (dc / 2 + 8) * 2.0 ** -24
    if cos is not None:
        err[:, dc:] += 3 * 2.0 ** -24 * (np.abs(y * cs) + oracle.rotate(np.abs(y), 0 * cs, np.abs(sn), inter).__abs__())
    if dtype == F16:
        err += 2.0 ** -25  # (below the smallest normal number)
    for t, s in enumerate(slots.tolist()):
        if 0 <= s < P * page:
            want[s], tol[s] = rows[t], err[t]
    d = np.abs(f64(cache).reshape(P * page, -1) - want)
    assert (d <= tol).all(), (np.argwhere(d > tol)[:3], d.max())
    assert (got is None) == (q is None)
    if q is not None:
        z = f64(q)
        ref = z if cos is None else oracle.rotate(z, cs[:, None], sn[:, None], inter)
        tq = np.abs(ref) * u * 1.01 + (2.0 ** -25 if dtype == F16 else 0)
        if cos is not None:
            tq = tq + 3 * 2.0 ** -24 * (np.abs(z * cs[:, None]) + np.abs(oracle.rotate(np.abs(z), 0 * cs[:, None], np.abs(sn[:, None]), inter)))
        assert (np.abs(f64(got) - ref) <= tq).all()


def test_append_in_place_queries_and_flat_cache(gpu):
    """q_out == q_pe at the C entry, rows [S, d], int32 slots, far rows of a strided cache."""
    from diffspec_mi355x import _ext
    T, dc, dr, H, S = 20, 256, 64, 4, 64
    c, pe = torch.randn((T, dc), device=gpu).to(BF), torch.randn((T, dr), device=gpu).to(BF)
    wide = torch.zeros((S, dc + dr + 64), dtype=BF, device=gpu)
    cache = wide[:, :dc + dr]
    slots = torch.randperm(S, device=gpu)[:T].int()
    cos, sin = tables(T, dr, False)
    q = torch.randn((T, H, dr), device=gpu).to(BF)
    want_q = append_latent_kv(c, pe, cache, slots, cos=cos, sin=sin, q_pe=q)
    first = wide.clone()
    wide.zero_()
    lib = _ext.load()
    _ext.check(lib.dsv_latent_append(_ext.desc(c), _ext.desc(pe), _ext.desc(None), 0.0, _ext.desc(cos), _ext.desc(sin), _ext.desc(None),
                                     0, _ext.desc(slots), _ext.desc(cache), _ext.desc(q), _ext.desc(q), _ext.stream_of(gpu)), "append")
    assert torch.equal(q, want_q) and torch.equal(wide, first)
    assert torch.equal(cache[slots.long(), :dc], c) and (wide[:, dc + dr:] == 0).all()


def test_append_of_no_tokens(gpu):
    cache = torch.ones((4, 8, 96), dtype=BF, device=gpu)
    m = token_slots(torch.zeros((1, 2), dtype=torch.int32, device=gpu), torch.zeros(1, dtype=torch.int32, device=gpu),
                    torch.zeros(1, dtype=torch.int32, device=gpu), 8, 0)
    none = lambda *s: torch.empty(s, dtype=BF, device=gpu)  # noqa: E731
    assert append_latent_kv(none(0, 64), none(0, 32), cache, m["slots"], q_pe=none(0, 4, 32)).shape == (0, 4, 32)
    assert append_latent_kv(none(0, 64), none(0, 32), cache, m["slots"]) is None
    assert (cache == 1).all()


def test_append_captured(gpu):
    """A captured append reads its slots and positions anew at every replay."""
    c, pe = torch.randn((30, 512), device=gpu).to(BF), torch.randn((30, 64), device=gpu).to(BF)
    cache = torch.zeros((8, 8, 576), dtype=BF, device=gpu)
    slots, pos = torch.randperm(64, device=gpu)[:30], torch.arange(30, device=gpu)
    cos, sin = tables(100, 64, False)
    q = torch.randn((30, 4, 64), device=gpu).to(BF)
    args = dict(cos=cos, sin=sin, positions=pos, q_pe=q)
    append_latent_kv(c, pe, cache, slots, **args)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = append_latent_kv(c, pe, cache, slots, **args)
    for i in range(3):
        cache.fill_(3)
        slots.copy_(torch.randperm(64, device=gpu)[:30])
        pos += i
        graph.replay()
        torch.cuda.synchronize()
        replayed = cache.clone()
        cache.fill_(3)
        want = append_latent_kv(c, pe, cache, slots, **args)
        assert torch.equal(got, want) and torch.equal(replayed, cache), i


@pytest.mark.parametrize("dtype", [BF, F32])
def test_decoding_loop(gpu, dtype):
    """Prompts expanded, their rows appended, then steps of extend, slots, append and absorbed attention over a forked
    and compacted pool: every step against attention over all tokens so far."""
    L, page, dc, dr, H, dn = 3, 16, 256, 64, 4, 64
    D, P, B, n_log = dc + dr, 60, 6, 16
    g = torch.Generator(device="cuda").manual_seed(0)
    rnd = lambda *s: torch.randn(s, generator=g, device=gpu).to(dtype)  # noqa: E731
    pool = torch.zeros((L, P, page, D), dtype=dtype, device=gpu)
    halves = pool.view(L, P, page, 2, D // 2).permute(0, 3, 1, 2, 4).unsqueeze(3)  # [L, 2, P, 1, page, D / 2]
    table = torch.full((B, n_log), -1, dtype=torch.int32, device=gpu)
    ref = torch.zeros(P, dtype=torch.int32, device=gpu)
    lens = torch.zeros(B, dtype=torch.int32, device=gpu)
    w_k, w_v = rnd(H, dn, dc).float() / math.sqrt(dc), rnd(H, dn, dc).float() / math.sqrt(dc)
    scale = (dn + dr) ** -0.5
    history = {0: [], 2: [], 4: []}     # sequence -> rows of layer 1
    layer = 1

    def step(seqs, new, cap):
        goal = lens.clone()
        goal[torch.tensor(seqs, device=gpu)] += torch.tensor(new, dtype=torch.int32, device=gpu)
        assert extend_pages(table, ref, lens, goal, page)[1:].tolist() == [0, 0]
        m = token_slots(table, lens, torch.tensor(new, dtype=torch.int32, device=gpu), page, cap,
                        seqs=torch.tensor(seqs, dtype=torch.int32, device=gpu))
        c, pe = rnd(cap, dc), rnd(cap, dr)
        before = pool[layer - 1].clone()
        append_latent_kv(c, pe, pool[layer], m["slots"])
        assert torch.equal(before, pool[layer - 1])
        rows, at = torch.cat([c, pe], 1), m["cu_seqlens"].tolist()
        for i, s in enumerate(seqs):
            history[s].append(rows[at[i]:at[i + 1]])
        return m

    # Prompts: the expanded form over the expanded rows equals the absorbed form, its output expanded.
    seqs, new = [4, 0, 2], [37, 20, 61]
    m = step(seqs, new, 128)
    q = rnd(len(seqs), max(new), H, dn + dr)
    absorbed = torch.cat([torch.einsum("bmhd,hdc->bmhc", q[..., :dn].float(), w_k), q[..., dn:].float()], -1).to(F32)
    N = max(new)
    dense = torch.zeros((3, N, D), device=gpu)
    for i, s in enumerate(seqs):
        dense[i, :new[i]] = history[s][0].float()
    k = torch.einsum("bnc,hdc->bnhd", dense[..., :dc], w_k).contiguous()
    v = torch.einsum("bnc,hdc->bnhd", dense[..., :dc], w_v).contiguous()
    e_out, e_lse = latent_attn_expanded(q.float(), k, dense[..., dc:], v, cache_seqlens=m["lens"], return_softmax_lse=True)
    a_out, a_lse = latent_attn_with_kvcache(absorbed, pool[layer].float(), dc, scale, cache_seqlens=m["lens"],
                                            page_table=m["block_table"], return_softmax_lse=True)
    torch.testing.assert_close(a_lse, e_lse, rtol=1e-4, atol=1e-4)
    torch.testing.assert_close(torch.einsum("bmhc,hdc->bmhd", a_out, w_v), e_out, rtol=1e-3, atol=1e-4)
    # A continuation of sequence 2 as sequence 1, then the pool is compacted.
    i32 = lambda *x: torch.tensor(x, dtype=torch.int32, device=gpu)  # noqa: E731
    assert fork_pages(halves, table, ref, lens, i32(2), i32(1))[1:].tolist() == [0, 0]
    history[1] = list(history[2])
    for it in range(4):
        if it == 2:
            compact_pages(halves, table, ref)
        seqs = [1, 2, 0, 4] if it % 2 else [4, 1, 2]
        new = [1] * len(seqs) if it != 1 else [3] * len(seqs)
        m = step(seqs, new, 16)
        q = rnd(len(seqs), new[0], H, D)
        out, lse = latent_attn_with_kvcache(q, pool[layer], dc, 0.06, cache_seqlens=m["lens"], page_table=m["block_table"],
                                            return_softmax_lse=True)
        u = torch.finfo(dtype).eps
        for i, s in enumerate(seqs):
            x = f64(torch.cat(history[s]))
            assert len(x) == int(m["lens"][i])
            for h in range(H):
                ref_ = oracle.attention(f64(q[i, :, h]), x, x[:, :dc], 0.06, oracle.visible(new[0], len(x)))
                tol = ref_["mass"] * (u + 1e-4) + u * np.abs(ref_["out"])
                assert (np.abs(f64(out[i, :, h]) - ref_["out"]) <= tol).all(), (it, s, h)
                assert np.abs(f64(lse[i, h]) - ref_["lse"]).max() <= 1e-4
