"""Page operations of a paged KV cache on MI355X: fork, extend, free, compact, slot maps.

The reference's ``PagedKVCache`` (``diffspec/core/kv_cache/paged_kv.py``) keeps
allocation, sharing and defragmentation in host code (:81-166, :364-402).
Here the bookkeeping lives on the device, so that a serving loop needs no host
round trip:

  * ``kv_pages``   [L, 2, P, Hk, page_size, D], the pool (:56-65);
  * ``page_table`` [B, n_logical] int32, each sequence's physical pages (-1:
    none), the form that ``tree_verify``, ``window_attn_with_kvcache``,
    ``append_tree_kv`` and ``kv_commit`` read;
  * ``refcount``   [P] int32, how many table entries name a page (0 = free);
  * ``seqlens``    [B] int32/int64, the tokens of each sequence.

``token_slots`` reads them: where the tokens of a step's requests stand in the
pool.  The other four calls change these tensors in place.  Pages are taken lowest first,
for requests in ascending order.  ``fork_pages`` and ``extend_pages`` either do
all that is asked or change nothing; the int32 tensor they return holds
(pages taken, pages lacking, requests refused), which a caller may read when
it next synchronises anyway.
"""

from __future__ import annotations

from typing import Dict, Optional

import torch

from ... import _ext

__all__ = ["fork_pages", "extend_pages", "free_pages", "compact_pages", "token_slots"]


def _page_ws(lib, refcount: torch.Tensor, page_table: torch.Tensor, n: int, dev) -> torch.Tensor:
    return _ext.workspace(lib.dsv_pages_workspace_bytes(refcount.numel(), page_table.shape[0], n), dev)


def fork_pages(kv_pages: torch.Tensor, page_table: torch.Tensor, refcount: torch.Tensor, seqlens: torch.Tensor,
               parents: torch.Tensor, children: torch.Tensor) -> torch.Tensor:
    """Sequence ``children[i]`` becomes a continuation of ``parents[i]``.

    Whole pages are shared (their counts grow); a partly filled last page is
    copied, in every layer, into a page of the child's own.  A parent may be
    named several times.  Refused (and then nothing is done): indices out of
    range, a child that is not empty (``seqlens != 0``; its row is overwritten, so
    free it first), that is named twice or that is a parent of the same call.

    Returns the int32 [3] tensor (pages taken, pages lacking, pairs refused).
    """
    dev = _ext.require_gpu(kv_pages, page_table, refcount, seqlens, parents, children)
    lib = _ext.load()
    with _ext.on_device(dev):
        info = torch.empty(3, dtype=torch.int32, device=dev)
        ws = _page_ws(lib, refcount, page_table, parents.numel(), dev)
        rc = lib.dsv_pages_fork(_ext.desc(kv_pages), _ext.desc(page_table), _ext.desc(refcount), _ext.desc(seqlens),
                                _ext.desc(parents), _ext.desc(children), _ext.desc(info), ws.data_ptr(), ws.numel(),
                                _ext.stream_of(dev))
    _ext.check(rc, "fork_pages")
    return info


def extend_pages(page_table: torch.Tensor, refcount: torch.Tensor, seqlens: torch.Tensor, new_lens: torch.Tensor,
                 page_size: int) -> torch.Tensor:
    """Grow sequences to ``new_lens`` [B] tokens; shorter or equal lengths change nothing.

    Pages that a sequence's row already names behind its ``seqlens`` are used
    before any is taken: a caller may set ``seqlens`` back after drafted tokens
    were rejected, and the next draft finds their pages.  (Not below tokens that
    it shares with another sequence: the pages are the other's too.)

    Returns the int32 [3] tensor (pages taken, pages lacking, sequences refused:
    new lengths that the table row cannot hold).
    """
    dev = _ext.require_gpu(page_table, refcount, seqlens, new_lens)
    lib = _ext.load()
    with _ext.on_device(dev):
        info = torch.empty(3, dtype=torch.int32, device=dev)
        ws = _page_ws(lib, refcount, page_table, 0, dev)
        rc = lib.dsv_pages_extend(_ext.desc(page_table), _ext.desc(refcount), _ext.desc(seqlens), _ext.desc(new_lens),
                                  _ext.i64(page_size), _ext.desc(info), ws.data_ptr(), ws.numel(), _ext.stream_of(dev))
    _ext.check(rc, "extend_pages")
    return info


def free_pages(page_table: torch.Tensor, refcount: torch.Tensor, seqlens: torch.Tensor, seqs: torch.Tensor,
               page_size: int, window: Optional[int] = None, sinks: int = 0) -> None:
    """Give pages of the sequences ``seqs`` [n] back.

    Without ``window`` all of them, and the sequences' lengths become 0.  With
    ``window`` (and ``sinks``) only the pages whose tokens no later token sees
    through a sliding window of that many tokens (``window_attn_with_kvcache``
    with the same arguments); lengths stay.  Entries of ``seqs`` out of range
    are skipped.
    """
    if window is not None and window < 1:
        raise ValueError(f"window must be at least 1 token (got {window})")
    dev = _ext.require_gpu(page_table, refcount, seqlens, seqs)
    lib = _ext.load()
    with _ext.on_device(dev):
        rc = lib.dsv_pages_free(_ext.desc(page_table), _ext.desc(refcount), _ext.desc(seqlens), _ext.desc(seqs),
                                _ext.i64(page_size), _ext.i64(window or 0), _ext.i64(sinks), _ext.stream_of(dev))
    _ext.check(rc, "free_pages")


def compact_pages(kv_pages: torch.Tensor, page_table: torch.Tensor, refcount: torch.Tensor) -> torch.Tensor:
    """Move the n pages in use to places [0, n), contents, counts and tables alike.

    Returns the int32 [3] tensor (pages in use, pages moved, 0).
    """
    dev = _ext.require_gpu(kv_pages, page_table, refcount)
    lib = _ext.load()
    with _ext.on_device(dev):
        info = torch.empty(3, dtype=torch.int32, device=dev)
        ws = _page_ws(lib, refcount, page_table, 0, dev)
        rc = lib.dsv_pages_compact(_ext.desc(kv_pages), _ext.desc(page_table), _ext.desc(refcount), _ext.desc(info),
                                   ws.data_ptr(), ws.numel(), _ext.stream_of(dev))
    _ext.check(rc, "compact_pages")
    return info


def token_slots(page_table: torch.Tensor, seqlens: torch.Tensor, new_lens: torch.Tensor, page_size: int, capacity: int,
                seqs: Optional[torch.Tensor] = None) -> Dict[str, torch.Tensor]:
    """Block tables and slot maps of a step's requests, built on the device.

    Request ``i`` is sequence ``seqs[i]`` (int32/int64 [n]; None: request ``i`` is
    sequence ``i``), whose last ``new_lens[i]`` of ``seqlens`` tokens are new
    (``extend_pages`` has given them pages).  In place of the reference's per-token host
    bookkeeping (``PagedKVCache.write_kv``, paged_kv.py:168-223).

    Args:
        capacity: tokens that the lists hold, whatever the lengths (which the host need
            not know); tokens beyond it are left out.

    Returns a dict:
        slots [capacity] int64: the new tokens' places, page * page_size + offset, in
            request order (-1 where the table names no page and behind the last token),
            as ``append_latent_kv`` takes them;
        positions, requests [capacity] int32: their positions and requests (-1 behind
            the last);
        cu_seqlens [n + 1] int32: where each request's tokens begin;
        block_table [n, n_logical] int32 and lens [n] int32: the requests' page lists
            (-1 behind their lengths) and lengths, as the attention calls take them.
    """
    dev = _ext.require_gpu(page_table, seqlens, new_lens, seqs)
    if page_table.dim() != 2:
        raise ValueError(f"page_table must be [B, n_logical] (got {tuple(page_table.shape)})")
    if not 0 <= int(capacity) <= 1 << 30:
        raise ValueError(f"capacity must be in [0, 2^30] (got {capacity})")
    n, cap, width = new_lens.numel(), int(capacity), page_table.shape[1]
    lib = _ext.load()
    with _ext.on_device(dev):
        # One allocation for all the lists (six take twice as long as the kernel).
        sizes = [2 * cap, cap, cap, n + 1, n * width, n]
        buf = torch.empty(sum(sizes), dtype=torch.int32, device=dev)
        slots, positions, requests, cu, block, lens = buf.split(sizes)
        at, out = buf.data_ptr(), []
        for size, dtype, shape in zip(sizes, (_ext.DSV_I64,) + 5 * (_ext.DSV_I32,),
                                      ((cap,), (cap,), (cap,), (n + 1,), (n, width), (n,))):
            out.append(_ext.desc_flat(at, dtype, *shape))
            at += 4 * size
        rc = lib.dsv_token_slots(_ext.desc(page_table), _ext.desc(seqlens), _ext.desc(new_lens), _ext.desc(seqs),
                                 _ext.i64(page_size), *out, _ext.stream_of(dev))
    _ext.check(rc, "token_slots")
    return {"slots": slots.view(torch.int64), "positions": positions, "requests": requests, "cu_seqlens": cu,
            "block_table": block.view(n, width), "lens": lens}
