"""Frequencies of rotary positions, plain or scaled for contexts longer than the trained one.

``rotary_frequencies`` gives what ``ops.rotary_append`` and ``ops.rotary_embedding`` take: the radians per position of
every pair, in 64 bits, and the factor that multiplies cosine and sine.
"""
from __future__ import annotations

import math

import torch


def rotary_frequencies(rot_dim: int, base: float = 10000.0, scaling: str | None = None, factor: float = 1.0,
                       original_max_position: int | None = None, fast_turns: float = 32.0, slow_turns: float = 1.0,
                       device=None):
    """-> (inv_freq float64 [rot_dim / 2], attention_factor).

    ``scaling``, for contexts ``factor`` times as long as the trained one:

    * ``None``      inv_freq[i] = base^(-2i / rot_dim);
    * ``"linear"``  every frequency divided by ``factor`` (position interpolation);
    * ``"ntk"``     the base raised to base * factor^(rot_dim / (rot_dim - 2)): the fastest pair keeps its frequency, the
      slowest is divided by ``factor``;
    * ``"yarn"``    pairs that turn more than ``fast_turns`` times over ``original_max_position`` positions keep their
      frequency, those that turn less than ``slow_turns`` times are divided by ``factor``, with a ramp that is linear in
      the pair's index between; attention_factor = 1 + ln(factor) / 10.
    """
    if rot_dim < 16 or rot_dim > 128 or rot_dim % 16:
        raise ValueError("rotary_frequencies: rot_dim must be a multiple of 16, at most 128")
    if not base > 1 or not factor >= 1:
        raise ValueError("rotary_frequencies: base must be above 1 and factor at least 1")
    i = torch.arange(rot_dim // 2, dtype=torch.float64)
    if scaling == "ntk":
        base = base * factor ** (rot_dim / (rot_dim - 2))
    inv_freq, attention_factor = base ** (-2 * i / rot_dim), 1.0
    if scaling == "linear":
        inv_freq = inv_freq / factor
    elif scaling == "yarn":
        if not original_max_position or original_max_position < 1 or not fast_turns > slow_turns > 0:
            raise ValueError("rotary_frequencies: yarn needs original_max_position and fast_turns > slow_turns > 0")
        # index of the pair that makes n turns over the trained context
        at = lambda n: rot_dim * math.log(original_max_position / (2 * math.pi * n)) / (2 * math.log(base))
        low = max(0, math.floor(at(fast_turns)))
        high = math.ceil(at(slow_turns))       # behind the last pair when even that one makes more than slow_turns turns
        slow = ((i - low) / (high - low)).clamp(0, 1) if high > low else (i >= high).double()
        inv_freq = inv_freq * (1 - slow) + inv_freq / factor * slow
        attention_factor = 1 + 0.1 * math.log(factor)
    elif scaling not in (None, "ntk"):
        raise ValueError(f"rotary_frequencies: unknown scaling {scaling!r}")
    return inv_freq.to(device) if device is not None else inv_freq, attention_factor
