"""Attention over a cache of one latent vector per token (gfx950 kernels of libdsv.so).

For target models whose cache row is a latent vector that all heads share and a
small rotated key part.  Two forms of one attention:

  * ``latent_attn_with_kvcache`` (absorbed): queries already in the latent space,
    over the cache itself; single tokens, drafted trees and chunks.  The contract is
    that of ``flash_attn_with_kvcache`` (the reference's
    ``diffspec/runtime/attention_compat.py:103-132``) with a page table and a tree;
  * ``latent_attn_expanded``: keys and values per head, as the expansion of the
    latent rows gives them; prompts.  Per (row, key) it needs about a third of the
    absorbed form's operations, and the expansion once per key.

Partial attentions over disjoint keys (a prompt's chunk over its cached prefix, and
over itself) join by their ``lse``.  There is no CPU path.
"""

from __future__ import annotations

from typing import Optional, Union

import torch

from .. import _ext

__all__ = ["latent_attn_with_kvcache", "latent_attn_expanded"]


def _lengths(cache_seqlens, B: int, cap: int):
    """(lengths per sequence or None, keys of every sequence)."""
    if isinstance(cache_seqlens, torch.Tensor):
        lens = cache_seqlens
        if lens.dim() == 0:
            lens = lens.reshape(1).expand(B)
        if lens.dtype not in (torch.int32, torch.int64):
            raise TypeError(f"cache_seqlens must be int32 or int64 (got {lens.dtype})")
        return lens.contiguous(), cap
    if cache_seqlens is None:
        return None, cap
    if int(cache_seqlens) < 0:
        raise ValueError(f"cache_seqlens must be >= 0 (got {cache_seqlens})")
    return None, min(int(cache_seqlens), cap)


def latent_attn_with_kvcache(q: torch.Tensor, kv_cache: torch.Tensor, v_dim: int, softmax_scale: float,
                             cache_seqlens: Optional[Union[int, torch.Tensor]] = None,
                             page_table: Optional[torch.Tensor] = None, parent: Optional[torch.Tensor] = None,
                             return_softmax_lse: bool = False, out_dtype: Optional[torch.dtype] = None):
    """Absorbed latent attention of the last M tokens of every sequence over its cache.

    A cache row is the key of every head and its first ``v_dim`` entries the value of
    every head.  Query m sees the keys up to its own token or, with ``parent``, the
    tokens before the tree, its ancestors and itself.  A query without a key returns
    zeros and ``-inf``.  M is one number for all sequences: one with fewer new tokens has
    them in its last rows, and the rows before them are for the caller to leave out.

    Scores and sums are float32; of 16-bit inputs the weights are rounded to their type
    before they meet the values, whatever ``out_dtype``.

    Args:
        q: [B, M, H, v_dim + dr] bf16/f16/f32: the queries times the key expansion, then
            their rotated part; v_dim 256 or 512, dr 32 or 64.
        kv_cache: dense [B, N, v_dim + dr], or pages [P, page_size, v_dim + dr] with
            ``page_table`` ([n_pages] or [B, n_pages] int32/int64).
        softmax_scale: of the model (1 / sqrt of the expanded query width, as a rule).
        cache_seqlens: tokens of each sequence, the M new ones included: an int or an
            int32/int64 [B] tensor; None: all that the cache holds.  Clamped to the cache.
        parent: [M] or [B, M] int32/int64 parent of each tree node (< 0: root),
            M <= 1024, as ``tree_verify``.

    Returns:
        out [B, M, H, v_dim] (``out_dtype``, default q's; still to be multiplied by the value
        expansion) and, if asked, lse [B, H, M] float32.
    """
    lens = cache_seqlens if isinstance(cache_seqlens, torch.Tensor) else None
    dev = _ext.require_gpu(q, kv_cache, lens, page_table, parent)
    if q.dim() != 4 or kv_cache.dim() != 3:
        raise ValueError(f"q must be 4-d and kv_cache 3-d (got {tuple(q.shape)} and {tuple(kv_cache.shape)})")
    if page_table is not None and page_table.dim() not in (1, 2):
        raise ValueError(f"page_table must be [n_pages] or [B, n_pages] (got {tuple(page_table.shape)})")
    B, M, H, _ = q.shape
    v_dim = int(v_dim)
    if not 1 <= v_dim <= q.shape[3]:
        raise ValueError(f"v_dim must be in [1, {q.shape[3]}] (got {v_dim})")
    cap = kv_cache.shape[1] if page_table is None else page_table.shape[-1] * kv_cache.shape[1]
    lib = _ext.load()
    with _ext.on_device(dev):
        lens, n = _lengths(cache_seqlens, B, cap)
        out = torch.empty((B, M, H, v_dim), dtype=out_dtype or q.dtype, device=dev)
        lse = torch.empty((B, H, M), dtype=torch.float32, device=dev) if return_softmax_lse else None
        q_d = _ext.desc(q)
        n_ws = lib.dsv_latent_workspace_bytes(B, M, H, v_dim, q_d.dtype, n, int(parent is not None), 0)
        ws, ws_ptr = _ext.scratch(n_ws, dev)
        rc = lib.dsv_latent_attention(q_d, _ext.desc(kv_cache), v_dim, _ext.desc(page_table), _ext.desc(lens), n,
                                      float(softmax_scale), _ext.desc(parent), _ext.desc(out), _ext.desc(lse), ws_ptr, n_ws,
                                      _ext.stream_of(dev))
    _ext.check(rc, "latent_attn_with_kvcache")
    return (out, lse) if return_softmax_lse else out


def latent_attn_expanded(q: torch.Tensor, k: torch.Tensor, k_pe: torch.Tensor, v: torch.Tensor,
                         softmax_scale: Optional[float] = None, cache_seqlens: Optional[Union[int, torch.Tensor]] = None,
                         causal: bool = True, return_softmax_lse: bool = False, out_dtype: Optional[torch.dtype] = None):
    """Expanded latent attention: keys and values per head, the rotated key part shared.

    Args:
        q: [B, M, H, dn + dr] bf16/f16/f32; dn 64 or 128, dr 32 or 64.
        k, v: [B, N, H, dn], for example the two halves of the expansion's output
            (any strides of whole 16 bytes).
        k_pe: [B, N, dr].
        softmax_scale: default 1 / sqrt(dn + dr).
        cache_seqlens: keys of each sequence (as ``latent_attn_with_kvcache``).
        causal: query m sees the keys n <= len - M + m, else all of its sequence.

    Returns:
        out [B, M, H, dn] (``out_dtype``, default q's) and, if asked, lse [B, H, M] float32.
        A query without a key gets zeros and ``-inf``.  Scores and sums are float32; of
        16-bit inputs the weights are rounded to their type before they meet the values.
    """
    lens = cache_seqlens if isinstance(cache_seqlens, torch.Tensor) else None
    dev = _ext.require_gpu(q, k, k_pe, v, lens)
    if q.dim() != 4 or k.dim() != 4 or v.dim() != 4:
        raise ValueError(f"q, k and v must be 4-d (got {tuple(q.shape)}, {tuple(k.shape)} and {tuple(v.shape)})")
    B, M, H, D = q.shape
    scale = D ** -0.5 if softmax_scale is None else float(softmax_scale)
    lib = _ext.load()
    with _ext.on_device(dev):
        lens, n = _lengths(cache_seqlens, B, k.shape[1])
        out = torch.empty((B, M, H, v.shape[3]), dtype=out_dtype or q.dtype, device=dev)
        lse = torch.empty((B, H, M), dtype=torch.float32, device=dev) if return_softmax_lse else None
        q_d = _ext.desc(q)
        n_ws = lib.dsv_latent_workspace_bytes(B, M, H, v.shape[3], q_d.dtype, n, 0, 1)
        ws, ws_ptr = _ext.scratch(n_ws, dev)
        rc = lib.dsv_latent_expanded(q_d, _ext.desc(k), _ext.desc(k_pe), _ext.desc(v), _ext.desc(lens), n, int(bool(causal)),
                                     scale, _ext.desc(out), _ext.desc(lse), ws_ptr, n_ws, _ext.stream_of(dev))
    _ext.check(rc, "latent_attn_expanded")
    return (out, lse) if return_softmax_lse else out
