"""Attention of one new token per sequence over a paged cache, through a block table.

Beside ``gqa_decode`` (32 query heads, 8 KV heads, head size 128, bf16, a list of whole pages): any number of
query heads per KV head, head sizes 64, 128 and 256, bf16 and fp16, e4m3 caches, a last page that is not full,
a sliding window.
"""
from . import _cabi


def run(q, k_cache, v_cache, block_table, seq_lens, sm_scale, k_scale=None, v_scale=None, window=0):
    """``q`` [batch, q_heads, dim]; caches [pages, page_size, kv_heads, dim] of q's type, or e4m3 with fp32 scales
    [pages, page_size, kv_heads] (``qk_norm_rope.run_to_cache`` writes both); token t of sequence b in page
    ``block_table[b, t // page_size]`` (int32), slot ``t % page_size``; ``seq_lens`` int32 [batch] with the new token
    counted in; ``window`` > 0: only the last so many tokens are visible.
    Any strides of the caches of whole 16 bytes with a contiguous last dimension will do.

    Returns (o like q, lse fp32 [batch, q_heads], the base-2 log of the sum of exp(sm_scale q.k)). A sequence that
    sees nothing gives o = 0, lse = -inf; tokens whose page id is outside the cache are not visible, and what lies there, or
    behind a sequence, does not matter. A visible key that scores minus infinity weighs 0 like one that is not visible, but 0
    times an infinite value, or a NaN, is NaN. bf16 queries over an e4m3 cache: elements of q that are 2^31 times smaller
    than the largest of their head lose bits (2^-39 of that)."""
    return _cabi.native().paged_decode(q, k_cache, v_cache, block_table, seq_lens, sm_scale, k_scale, v_scale, window)
