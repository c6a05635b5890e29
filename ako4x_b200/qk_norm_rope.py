"""The RMS norm of every query and key head with the rotation of ``rope`` in the same pass, and with keys
and values stored into a paged cache.

``x * rsqrt(mean(x^2) + eps) * weight`` over each head, then the rotation; fp32 in between, rounded once. Shapes,
types and strides of ``q``, ``k``, ``positions`` and ``inv_freq`` as in ``rope.run``; weights [dim], of the rows' type
or fp32.
"""
from . import _cabi


def run(q, k, q_weight, k_weight, positions, inv_freq, eps=1e-6, interleaved=False, attention_factor=1.0):
    """Returns (q_out, k_out), contiguous."""
    return _cabi.native().qk_norm_rope(q, k, q_weight, k_weight, positions, inv_freq, eps, interleaved, attention_factor)


def run_to_cache(q, k, v, q_weight, k_weight, positions, inv_freq, slot_mapping, k_cache, v_cache, k_scale=None,
                 v_scale=None, eps=1e-6, interleaved=False, attention_factor=1.0):
    """Returns q_out and stores the keys, and ``v`` as it is, at ``slot_mapping`` (page * page_size + slot, int32 or
    int64, distinct) of ``k_cache`` / ``v_cache`` [pages, page_size, k_heads, dim], in place. A slot outside the cache
    (-1) leaves that token out of it. A weight of None leaves that norm out: rotation and store alone.

    The caches are of the rows' type, or e4m3 with fp32 scales ``k_scale`` / ``v_scale`` [pages, page_size, k_heads],
    one per row: amax / 448, or 1 where amax <= 1e-10. Any strides of whole 16 bytes (e4m3: 8) with a contiguous
    last dimension will do."""
    return _cabi.native().qk_norm_rope_cache(q, k, v, q_weight, k_weight, positions, inv_freq, slot_mapping, k_cache, v_cache,
                                             k_scale, v_scale, eps, interleaved, attention_factor)
