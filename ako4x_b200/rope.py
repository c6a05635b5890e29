"""Rotary positions of queries and keys: half and interleaved pairs, part of the head, frequencies
scaled for long contexts.

``run(q, k, positions, inv_freq) -> (q_out, k_out)`` rotates the first ``2 * inv_freq.numel()`` elements of
every head of ``q`` [tokens, q_heads, dim] and ``k`` [tokens, k_heads, dim] (or None) by the angles
``positions * inv_freq`` and copies the rest; bf16 or fp16, ``dim`` a multiple of 8 up to 256, any token and
head strides (slices of one projection). Angles are taken in 64 bits, so far positions are as exact as
near ones. ``frequencies`` makes ``inv_freq``.
"""
import math

import torch

from . import _cabi


def run(q, k, positions, inv_freq, interleaved=False, attention_factor=1.0):
    """Pairs are (i, i + rotary_dim / 2), or (2i, 2i + 1) when ``interleaved``; cosine and sine are
    multiplied by ``attention_factor``. ``positions`` int32 or int64 [tokens], ``inv_freq`` fp32."""
    return _cabi.native().rope(q, k, positions, inv_freq, interleaved, attention_factor)


def frequencies(rotary_dim, base=10000.0, scaling="none", factor=1.0, original_length=None, beta_fast=32.0, beta_slow=1.0,
                device="cuda"):
    """``(inv_freq fp32 [rotary_dim / 2], attention_factor)``.

    ``scaling``: "none", ``base ** (-2i / rotary_dim)``; "linear", these divided by ``factor`` (positions
    interpolated); "ntk", the base raised so that the lowest frequency is divided by ``factor``; "yarn" (Peng et
    al., 2023), frequencies that turn more than ``beta_fast`` times in ``original_length`` tokens kept, those below
    ``beta_slow`` turns divided by ``factor``, a linear ramp over i between them, attention factor 0.1 ln(factor) + 1.
    """
    if rotary_dim < 2 or rotary_dim % 2:
        raise _cabi.Ako4xError("rope: rotary_dim must be even and positive")
    if not (base > 0 and factor > 0):
        raise _cabi.Ako4xError("rope: base and factor must be positive")
    half = rotary_dim // 2
    i = torch.arange(half, dtype=torch.float64)
    attention_factor = 1.0
    if scaling == "none":
        f = base ** (-i / half)
    elif scaling == "linear":
        f = base ** (-i / half) / factor
    elif scaling == "ntk":
        if half < 2:
            raise _cabi.Ako4xError("rope: ntk scaling needs rotary_dim >= 4")
        f = (base * factor ** (half / (half - 1))) ** (-i / half)
    elif scaling == "yarn":
        if original_length is None or original_length < 1:
            raise _cabi.Ako4xError("rope: yarn scaling needs original_length")
        if not base > 1:
            raise _cabi.Ako4xError("rope: yarn scaling needs a base above 1")
        if not beta_fast >= beta_slow > 0:
            raise _cabi.Ako4xError("rope: yarn scaling needs beta_fast >= beta_slow > 0")

        def index_of(turns):   # of the frequency that turns so often
            return half * math.log(original_length / (2 * math.pi * turns)) / math.log(base)

        low, high = max(math.floor(index_of(beta_fast)), 0), min(math.ceil(index_of(beta_slow)), rotary_dim - 1)
        ramp = ((i - low) / max(high - low, 1e-3)).clamp(0.0, 1.0)
        ramp[i > index_of(beta_slow)] = 1.0   # all of them, where the first one turns too seldom already
        f = base ** (-i / half) * (1.0 - ramp + ramp / factor)
        if factor > 1:
            attention_factor = 0.1 * math.log(factor) + 1.0
    else:
        raise _cabi.Ako4xError(f"rope: unknown scaling {scaling!r}")
    return f.to(torch.float32).to(device), attention_factor
