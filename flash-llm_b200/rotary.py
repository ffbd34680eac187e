"""Angles of rotary positions: the frequencies that ``rotary_append`` takes, for the usual ways to stretch a context."""
from __future__ import annotations

import math

import numpy as np


def rotary_frequencies(rotary_dim: int, base: float = 10000.0, scaling: str = "none", factor: float = 1.0,
                       original_length: int = 0, slow_turns: float = 1.0, fast_turns: float = 32.0) -> tuple[np.ndarray, float]:
    """``(frequencies float64[rotary_dim / 2], magnitude)``: radians per position of pair i, ``base ** (-2 i / rotary_dim)``
    before scaling, and the factor on the turned values.  ``scaling`` stretches a model's context by ``factor``:

    * ``"none"``;
    * ``"linear"``: positions are squeezed, every frequency divided by ``factor``;
    * ``"base"``: the base grows by ``factor ** (rotary_dim / (rotary_dim - 2))``, so that the slowest pair is slowed by
      ``factor`` and the fastest kept;
    * ``"by parts"``: pairs that turn more than ``fast_turns`` times over ``original_length`` positions are kept, those that turn
      less than ``slow_turns`` times are slowed by ``factor``, linearly in the turns between; the magnitude is
      ``0.1 ln(factor) + 1`` (the published YaRN method).
    """
    if rotary_dim <= 0 or rotary_dim % 16 != 0:
        raise ValueError(f"rotary_dim={rotary_dim} must be a positive multiple of 16")
    if not (base > 0 and math.isfinite(base)) or not (factor > 0 and math.isfinite(factor)):
        raise ValueError(f"base={base} and factor={factor} must be positive and finite")
    exponent = np.arange(0, rotary_dim, 2, dtype=np.float64) / rotary_dim
    if scaling == "base":
        base = base * factor ** (rotary_dim / (rotary_dim - 2))
    frequencies = base ** -exponent
    if scaling in ("none", "base"):
        return frequencies, 1.0
    if scaling == "linear":
        return frequencies / factor, 1.0
    if scaling == "by parts":
        if original_length <= 0 or not 0 <= slow_turns < fast_turns:
            raise ValueError("scaling by parts needs the original_length and slow_turns < fast_turns")
        keep = np.clip((original_length * frequencies / (2 * math.pi) - slow_turns) / (fast_turns - slow_turns), 0.0, 1.0)
        return frequencies * keep + frequencies / factor * (1 - keep), 0.1 * math.log(max(factor, 1.0)) + 1.0
    raise ValueError(f"unknown scaling {scaling!r}: none, linear, base or by parts")
