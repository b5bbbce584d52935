"""A step whose requests have different numbers of new tokens: packed rows, laid into those of the attention call."""

import numpy as np
import pytest
import torch

from diffspec_mi355x.core.kv_cache import token_slots
from diffspec_mi355x.runtime.cache_state import append_latent_kv
from diffspec_mi355x.runtime.latent_attention import latent_attn_with_kvcache
from oracle import latent as oracle
from test_gpu_latent import BF, F16, F32, check, f64

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [BF, F16, F32])
@pytest.mark.parametrize("new,old", [([3, 1, 7, 0, 2], [40, 0, 130, 9, 511]), ([1, 1, 1], [5, 6, 7]), ([20], [0])])
def test_mixed_new_lengths(gpu, dtype, new, old):
    page, H, dc, dr = 16, 3, 256, 64
    D, n, scale = dc + dr, len(new), 0.05
    g = torch.Generator(device="cuda").manual_seed(n)
    lens = [a + b for a, b in zip(new, old)]
    n_log = -(-max(lens) // page)
    perm = torch.from_numpy(np.random.default_rng(n).permutation(n * n_log).astype(np.int32))
    table = perm.view(n, n_log).to(gpu)
    pool = torch.randn((n * n_log, page, D), generator=g, device=gpu).to(dtype)
    cap, M = sum(new) + 3, max(new)
    m = token_slots(table, torch.tensor(lens, device=gpu), torch.tensor(new, device=gpu), page, cap)
    c, pe = (torch.randn((cap, w), generator=g, device=gpu).to(dtype) for w in (dc, dr))
    q_packed = torch.randn((cap, H, D), generator=g, device=gpu).to(dtype)
    append_latent_kv(c, pe, pool, m["slots"])

    r, pos = m["requests"].long(), m["positions"].long()
    row = (M - (m["lens"].long()[r] - pos)).clamp(0, M - 1)
    q = q_packed.new_zeros((n + 1, M, H, D))
    q[r, row] = q_packed
    out, lse = latent_attn_with_kvcache(q[:n], pool, dc, scale, m["lens"], m["block_table"], return_softmax_lse=True)
    packed = out[r, row]

    at = 0
    for i in range(n):
        x = f64(pool[table[i].long()].reshape(-1, D)[:lens[i]])
        rows = list(range(M - new[i], M))
        assert torch.equal(packed[at:at + new[i]], out[i, M - new[i]:])
        for t in range(new[i]):
            want = f64(torch.cat([c[at + t], pe[at + t]]))
            assert np.array_equal(x[old[i] + t], want)
        seen = [np.arange(old[i] + t + 1) for t in range(new[i])]
        for h in range(H):
            if new[i]:
                ref = oracle.attention(f64(q_packed[at:at + new[i], h]), x, x[:, :dc], scale, seen)
                check(out[:, rows], lse[:, :, rows], i, h, ref, D, dtype, lens[i], np.abs(x).max())
        at += new[i]
