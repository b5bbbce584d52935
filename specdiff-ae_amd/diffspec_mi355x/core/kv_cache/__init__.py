"""Paged KV cache: page operations on device tables (gfx950 kernels)."""

from .paged_kv import compact_pages, extend_pages, fork_pages, free_pages, token_slots  # noqa: F401
