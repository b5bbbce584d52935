"""diffspec_mi355x — MI355X-native (gfx950) tree-verification hot path of DiffSpec.

Module layout mirrors the reference package ``diffspec``:
  runtime.tree_attention     prefix_attention_forward, tree_attention_forward, tree_verify
  runtime.attention_compat   flash_attn_with_kvcache / flash_attn_func contract
  runtime.bundle_verifier    FusedBundleVerifier, PagedBundleVerifier
  core.bundle_scheduler      BundleScheduler, TreeDescriptorBuilder, bundle_row_order,
                             bundle_row_order_device
  runtime.window_attention   window_attn_with_kvcache
  runtime.latent_attention   latent_attn_with_kvcache, latent_attn_expanded
  runtime.cache_state        append_tree_kv, append_latent_kv
  core.kv_cache              fork_pages, extend_pages, free_pages, compact_pages, token_slots
  draft.tree_verification    verify / verify_new, tree_accept, speculative_accept, evaluate_tree
All compute runs in libdsv.so (HIP kernels for gfx950 behind a C ABI).
"""

__version__ = "0.1.0"
