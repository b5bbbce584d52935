"""Attention through a sliding window with a few first tokens that stay visible.

``flash_attn_with_kvcache`` (the reference's
``diffspec/runtime/attention_compat.py:103-132``) with a window, sinks, a page
table and an optional tree of drafted tokens: for models with windowed layers,
and for caches that keep the first and the recent tokens (the reference's draft
side keeps such a working cache, ``diffspec/draft/draft_network.py:1250-1331``).
The work is done by libdsv.so (``dsv_window_attention``); there is no CPU path.
"""

from __future__ import annotations

from typing import Optional, Union

import torch

from .. import _ext

__all__ = ["window_attn_with_kvcache"]


def window_attn_with_kvcache(q: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor, window: int,
                             sinks: int = 0, cache_seqlens: Optional[Union[int, torch.Tensor]] = None,
                             page_table: Optional[torch.Tensor] = None, parent: Optional[torch.Tensor] = None,
                             return_softmax_lse: bool = False, out_dtype: Optional[torch.dtype] = None):
    """Windowed attention of the last M tokens of every sequence over its cache.

    Query m of a sequence of ``len`` tokens has position ``p = len - M + m`` and
    sees the keys ``n <= p`` with ``n > p - window`` or ``n < sinks``.  With
    ``parent`` it is node m of a drafted tree whose keys are the cache's last M:
    ``p = len - M + depth(m)``, and of the tree it sees its ancestors and itself
    (each at its own depth's position).  A query without a key returns zeros and
    ``-inf``.

    Args:
        q: [B, M, H, D] bf16/f16/f32, D 64 or 128; one token (M = 1), a chunk of
            a prompt or a tree.
        k_cache, v_cache: dense [B, N, Hk, D], or page-pool halves
            [P, Hk, page_size, D] with ``page_table``; Hk divides H.
        window: tokens that a query sees up to its own, >= 1.
        sinks: first tokens of the sequence that stay visible.
        cache_seqlens: tokens of each sequence, the M new ones included: an int
            or an int32/int64 [B] tensor; None: all that the cache holds.
            Values are clamped to the cache.
        page_table: [n_pages] or [B, n_pages] int32/int64; pages that no query
            sees may be missing (-1), as ``free_pages(window=, sinks=)`` leaves them.
        parent: [M] or [B, M] int32/int64 parent of each tree node (< 0: root),
            M <= 1024, as ``tree_verify``.

    Returns:
        out [B, M, H, D] (``out_dtype``, default q's) and, if asked, lse [B, H, M]
        float32.
    """
    lens = cache_seqlens if isinstance(cache_seqlens, torch.Tensor) else None
    dev = _ext.require_gpu(q, k_cache, v_cache, lens, page_table, parent)
    if q.dim() != 4 or k_cache.dim() != 4:
        raise ValueError(f"q and the caches must be 4-d (got {tuple(q.shape)} and {tuple(k_cache.shape)})")
    B, M, H, D = q.shape
    if page_table is not None and page_table.dim() not in (1, 2):
        raise ValueError(f"page_table must be [n_pages] or [B, n_pages] (got {tuple(page_table.shape)})")
    if page_table is not None:
        Hk, cap = k_cache.shape[1], page_table.shape[-1] * k_cache.shape[2]
    else:
        Hk, cap = k_cache.shape[2], k_cache.shape[1]
    n, window, sinks = cap, _ext.i64(window), _ext.i64(sinks)
    if lens is not None:
        if lens.dim() == 0:
            lens = lens.reshape(1).expand(B).contiguous()
        if lens.dtype not in (torch.int32, torch.int64):
            raise TypeError(f"cache_seqlens must be int32 or int64 (got {lens.dtype})")
        lens = lens.contiguous()
    elif cache_seqlens is not None:
        if int(cache_seqlens) < 0:
            raise ValueError(f"cache_seqlens must be >= 0 (got {cache_seqlens})")
        n = min(int(cache_seqlens), cap)
    lib = _ext.load()
    with _ext.on_device(dev):
        out = torch.empty((B, M, H, D), dtype=out_dtype or q.dtype, device=dev)
        lse = torch.empty((B, H, M), dtype=torch.float32, device=dev) if return_softmax_lse else None
        q_d = _ext.desc(q)
        n_ws = lib.dsv_window_workspace_bytes(B, M, H, Hk, D, q_d.dtype, n, window, sinks, int(parent is not None))
        ws, ws_ptr = _ext.scratch(n_ws, dev)
        rc = lib.dsv_window_attention(q_d, _ext.desc(k_cache), _ext.desc(v_cache), _ext.desc(page_table),
                                      _ext.desc(lens), n, window, sinks, _ext.desc(parent), _ext.desc(out),
                                      _ext.desc(lse), ws_ptr, n_ws, _ext.stream_of(dev))
    _ext.check(rc, "window_attn_with_kvcache")
    return (out, lse) if return_softmax_lse else out
