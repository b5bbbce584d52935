"""fp32 latent attention: the sums of a score's products are short, so that a large one does not swallow the rest.

Sums of 64 products round at most 64 times, and D / 64 of them are added: a score is off by at most
(64 + D / 64 + 1) 2^-24 sum |q k|, a ninth to a half of what one chain of all D products may lose.  The logarithm of one
key's weight is its score; its own roundings (product with the scale, sum, product with ln 2) are 4 half steps."""

import pytest
import torch

from diffspec_mi355x.runtime.latent_attention import latent_attn_expanded, latent_attn_with_kvcache

pytestmark = pytest.mark.gpu


def bound(D, reach, scale):
    return (64 + D // 64 + 1 + 4) * 2.0 ** -24 * reach * scale


@pytest.mark.parametrize("dc,dr", [(512, 64), (512, 32), (256, 64)])
@pytest.mark.parametrize("M,H", [(1, 3), (2, 40)])
@pytest.mark.parametrize("at", [0, 70, 300, -1])
def test_absorbed(gpu, dc, dr, M, H, at):
    D, n, scale = dc + dr, M, 1 / 64
    if at >= dc:
        at = 100
    q = torch.full((1, M, H, D), 0.5, device=gpu)
    kv = torch.full((1, n, D), 0.5, device=gpu)
    q[..., at] = 4096.0
    kv[..., at] = 4096.0
    s = 2.0 ** 24 + 0.25 * (D - 1)
    _, lse = latent_attn_with_kvcache(q, kv, dc, scale, cache_seqlens=1 if M == 1 else None, return_softmax_lse=True)
    assert abs(float(lse[0, 0, 0]) - s * scale) <= bound(D, s, scale)
    assert (lse[0, :, 0] == lse[0, 0, 0]).all()


@pytest.mark.parametrize("dn,dr", [(128, 64), (64, 32)])
def test_expanded(gpu, dn, dr):
    D, scale = dn + dr, 1 / 64
    q, k, pe = (torch.full(x, 0.5, device=gpu) for x in ((1, 1, 2, D), (1, 1, 2, dn), (1, 1, dr)))
    q[..., 0] = k[..., 0] = 4096.0
    s = 2.0 ** 24 + 0.25 * (D - 1)
    _, lse = latent_attn_expanded(q, k, pe, k, softmax_scale=scale, return_softmax_lse=True)
    assert (lse.double() - s * scale).abs().max() <= bound(D, s, scale)
