"""Drafted trees over a latent pool: their rows appended, attended to, the accepted ones committed, and the next token's
attention over what stays."""

import numpy as np
import pytest
import torch

from diffspec_mi355x.core.kv_cache import extend_pages, token_slots
from diffspec_mi355x.draft.tree_verification import kv_commit
from diffspec_mi355x.runtime.cache_state import append_latent_kv
from diffspec_mi355x.runtime.latent_attention import latent_attn_with_kvcache
from oracle import latent as oracle
from test_gpu_latent import BF, F16, F32, chain_tree, compare, f64

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype,dc,dr,M,parts", [(BF, 512, 64, 40, 1), (F16, 256, 32, 64, 1), (F32, 512, 64, 30, 1),
                                                 (BF, 512, 64, 300, 4), (F32, 256, 32, 200, 3)])
def test_tree_rows_are_committed(gpu, dtype, dc, dr, M, parts):
    """The pool goes to kv_commit as halves of rows in the place of K and V, and parts of a half in that of heads, so that
    trees of more nodes fit what a workgroup holds.  Moved rows are equal bit for bit, others stay."""
    L, page, H, B, D = 2, 16, 3, 3, dc + dr
    rng = np.random.default_rng(M)
    g = torch.Generator(device="cuda").manual_seed(M)
    rnd = lambda *s: torch.randn(s, generator=g, device=gpu).to(dtype)  # noqa: E731
    prefix = [45, 0, 120]
    n_log = -(-(max(prefix) + M + 1) // page)
    P = B * n_log + 3
    pool = rnd(L, P, page, D)
    table = torch.full((B, n_log), -1, dtype=torch.int32, device=gpu)
    ref = torch.zeros(P, dtype=torch.int32, device=gpu)
    lens = torch.zeros(B, dtype=torch.int32, device=gpu)
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device=gpu)  # noqa: E731
    rows = [[torch.zeros((0, D), dtype=dtype, device=gpu)] * B for _ in range(L)]

    def step(new):
        assert extend_pages(table, ref, lens, lens + i32(new), page)[1:].tolist() == [0, 0]
        cap = sum(new) + 2
        m = token_slots(table, lens, i32(new), page, cap)
        at = m["cu_seqlens"].tolist()
        for x in range(L):
            c, pe = rnd(cap, dc), rnd(cap, dr)
            append_latent_kv(c, pe, pool[x], m["slots"])
            new_rows = torch.cat([c, pe], 1)
            rows[x] = [torch.cat([rows[x][b], new_rows[at[b]:at[b + 1]]]) for b in range(B)]

    def attend(n, parent=None):
        for x in range(L):
            q = rnd(B, n, H, D)
            out, lse = latent_attn_with_kvcache(q, pool[x], dc, 0.05, cache_seqlens=lens, page_table=table, parent=parent,
                                                return_softmax_lse=True)
            compare(q, rows[x], [len(r) for r in rows[x]], dc, 0.05, out, lse, parent, range(H), dtype)

    step(prefix)
    step([M] * B)
    attend(M, torch.tensor([chain_tree(rng, M) for _ in range(B)], device=gpu))
    # The walk's outputs: a path of each tree, one of a root alone.
    path = torch.full((B, M), -1, dtype=torch.int64)
    n = [1 + int(rng.integers(3, M // 2)), 1, M // 2]
    for b in range(B):
        p = np.concatenate([[0], np.sort(rng.choice(np.arange(1, M), n[b] - 1, replace=False))])
        path[b, :n[b]] = torch.from_numpy(p)
    info = torch.zeros((B, 4), dtype=torch.int64)
    info[:, 3] = torch.tensor(n)
    pd, idv = path.to(gpu), info.to(gpu)
    before = pool.clone()
    view = pool.view(L, P, page, 2, parts, D // 2 // parts).permute(0, 3, 1, 4, 2, 5)
    for b in range(B):
        kv_commit(view, prefix[b], pd, idv, page_table=table[b], tree=b)
        lens[b] = prefix[b] + n[b]
    want = before.view(L, P * page, D).clone()
    slot = lambda b, t: int(table[b, t // page]) * page + t % page  # noqa: E731
    for b in range(B):
        for i in range(n[b]):
            want[:, slot(b, prefix[b] + i)] = before.view(L, P * page, D)[:, slot(b, prefix[b] + int(path[b, i]))]
    assert torch.equal(pool.view(L, P * page, D), want)
    rows = [[torch.cat([r[b][:prefix[b]], r[b][prefix[b]:][path[b, :n[b]]]]) for b in range(B)] for r in rows]
    step([1] * B)
    attend(1)
