"""Latent attention over rows so far apart that their distances leave 32 bits, over pages longer than any sequence, and
over no keys at all."""

import pytest
import torch

from diffspec_mi355x.runtime.latent_attention import latent_attn_expanded, latent_attn_with_kvcache
from test_gpu_latent import BF, F16, F32, compare, compare_exp

pytestmark = pytest.mark.gpu

FAR = (1 << 24) + 24  # entries between two rows


def far_rows(g, dtype, *shape):
    """[1, N, ..] rows at distances of FAR entries."""
    n, rest = shape[0], shape[1:]
    size = 1
    for x in rest:
        size *= x
    buf = torch.empty((n - 1) * FAR + size, dtype=dtype, device="cuda")
    strides, at = [], 1
    for x in reversed(rest):
        strides.insert(0, at)
        at *= x
    t = buf.as_strided((1, n, *rest), (0, FAR, *strides))
    t.copy_(torch.randn((1, n, *rest), generator=g, device="cuda").to(dtype))
    return t


@pytest.mark.parametrize("dtype", [BF, F16, F32])
@pytest.mark.parametrize("M,H", [(1, 16), (3, 40), (40, 2)])
def test_absorbed_rows_far_apart(gpu, dtype, M, H):
    g = torch.Generator(device="cuda").manual_seed(M)
    n, dc, dr = 70, 256, 32
    kv = far_rows(g, dtype, n, dc + dr)
    q = torch.randn((1, M, H, dc + dr), generator=g, device=gpu).to(dtype)
    out, lse = latent_attn_with_kvcache(q, kv, dc, 0.06, return_softmax_lse=True)
    compare(q, [kv[0].contiguous()], [n], dc, 0.06, out, lse, None, range(H), dtype)
    # The same rows as pages of one token each (stride of a page).
    table = torch.randperm(n, generator=torch.Generator().manual_seed(1)).to(gpu)
    pages = kv.view(n, 1, dc + dr)
    out, lse = latent_attn_with_kvcache(q, pages, dc, 0.06, page_table=table, return_softmax_lse=True)
    compare(q, [kv[0][table]], [n], dc, 0.06, out, lse, None, range(H), dtype)


@pytest.mark.parametrize("dtype", [BF, F16, F32])
@pytest.mark.parametrize("M", [1, 40, 64])
@pytest.mark.parametrize("which", ["k", "v", "k_pe", "q"])
def test_expanded_rows_far_apart(gpu, dtype, M, which):
    g = torch.Generator(device="cuda").manual_seed(M)
    n, H, dn, dr = 70, 2, 64, 32
    make = lambda name, *s: (far_rows(g, dtype, *s) if name == which  # noqa: E731
                             else torch.randn((1, *s), generator=g, device=gpu).to(dtype))
    k, v, pe, q = make("k", n, H, dn), make("v", n, H, dn), make("k_pe", n, dr), make("q", M, H, dn + dr)
    out, lse = latent_attn_expanded(q, k, pe, v, return_softmax_lse=True)
    compare_exp(q, k, pe, v, [n], True, (dn + dr) ** -0.5, out, lse, range(H), dtype)


@pytest.mark.parametrize("dtype", [BF, F32])
def test_long_pages(gpu, dtype):
    g = torch.Generator(device="cuda").manual_seed(2)
    B, M, H, dc, D = 3, 2, 5, 512, 576
    pool = torch.randn((4, 8192, D), generator=g, device=gpu).to(dtype)
    table = torch.tensor([[2], [0], [3]], device=gpu)
    lens = [1, 900, 65]
    q = torch.randn((B, M, H, D), generator=g, device=gpu).to(dtype)
    out, lse = latent_attn_with_kvcache(q, pool, dc, 0.05, torch.tensor(lens, device=gpu), table, return_softmax_lse=True)
    compare(q, [pool[int(table[b]), :lens[b]] for b in range(B)], lens, dc, 0.05, out, lse, None, range(H), dtype)


@pytest.mark.parametrize("dtype", [BF, F16, F32])
def test_no_keys(gpu, dtype):
    """A length of 0 for all sequences, as a number: zeros and -inf, whatever the cache holds."""
    q = torch.randn((2, 3, 4, 288), device=gpu).to(dtype)
    kv = torch.full((2, 5, 288), float("nan"), dtype=dtype, device=gpu)
    out, lse = latent_attn_with_kvcache(q, kv, 256, 0.06, cache_seqlens=0, return_softmax_lse=True)
    assert (out == 0).all() and torch.isneginf(lse).all()
    k = torch.full((2, 5, 4, 64), float("nan"), dtype=dtype, device=gpu)
    for causal in (True, False):
        out, lse = latent_attn_expanded(q[..., :96].contiguous(), k, k[:, :, 0, :32], k, cache_seqlens=0, causal=causal,
                                        return_softmax_lse=True)
        assert (out == 0).all() and torch.isneginf(lse).all()
