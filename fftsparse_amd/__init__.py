"""fftsparse_amd -- MI355X-native FFTSparse prefill (FFT-guided block selection
+ block-sparse causal GQA attention) on hand-written gfx950 HIP kernels.

Public API (drop-in for attn_src/fft_attn/my_attn_v7.py and
attn_src/fix_mask_attn/my_attn.py):

    myattn_prefill(q, k, v, layer_idx, ...)        v7 selection + sparse attention
    fix_mask.myattn_prefill(q, k, v, layer_idx, ...) fixed sink/recent/local mask
    select_blocks(q, k, ...)                        stage 1 only (the block mask)
    block_sparse_attention(q, k, v, cnt, bits, ...) stage 2 only (or block_mask=: base_blockmask)
    rope_pool(q, k, cos, sin, ...)                  the rotary embedding before the call, fused
                                                    with the block pooling (select_blocks(pooled=...))

The reference's comparison selectors on the same attention kernel:

    xattn.Xattention_prefill(q, k, v, ...)          attn_src/xattn/src/Xattention.py
    flex.Flexprefill_prefill(q, k, v, ...)          attn_src/Flexprefill.py

Serving after the prefill, over a paged cache (no counterpart in the reference):

    plan_step(block_table, seq_lens, new_lens, ...) block tables and slot maps of a step, on the GPU
    rope(q, k, positions, inv_freq, ...)            rotary positions (rope_frequencies: plain or scaled)
    rope_cache(q, k, v, positions, slots, ...)      the same, keys and values into the cache
    paged_attention(q, k_cache, v_cache, ...)       new tokens (one or a chunk) over the cache
    plan_tree, tree_attention, accept_tree, move_kept   drafted tokens as a tree: attention, the path that is kept
    window_attention(q, k, v, window=, sinks=)      sliding window and first tokens, on contiguous K/V
"""
from .attn import (AttentionCall, BlockSelection, block_sparse_attention, myattn_prefill, rope_pool,  # noqa: F401
                   select_blocks)
from .paged import StepPlan, paged_attention, plan_step, window_attention  # noqa: F401
from .rotary import rope, rope_cache, rope_frequencies  # noqa: F401
from .tree import Accepted, TreePlan, accept_tree, move_kept, plan_tree, tree_attention  # noqa: F401
from . import fix_mask, flex, xattn  # noqa: F401

__all__ = ["myattn_prefill", "select_blocks", "block_sparse_attention", "rope_pool", "AttentionCall",
           "BlockSelection", "StepPlan", "plan_step", "rope", "rope_cache", "rope_frequencies", "paged_attention",
           "window_attention", "TreePlan", "plan_tree", "tree_attention", "Accepted", "accept_tree", "move_kept", "fix_mask", "flex", "xattn"]
