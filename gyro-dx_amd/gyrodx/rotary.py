"""Frequencies of rotary positions, for Engine.add_rotary."""
import math

import numpy as np

SCALINGS = ("none", "linear", "base", "bands")


def frequencies(dim: int, base: float = 10000.0, scaling: str = "none", factor: float = 1.0, context: int = 4096,
                slow: float = 1.0, fast: float = 32.0):
    """(float64 [dim / 2] frequencies in radians per position, scale of the turned values) for the first `dim` values of a head.

    Unscaled, pair j turns by base^(-2 j / dim) a position. For contexts `factor` times the one of `context` positions that
    a model was trained on:
      linear  every position is divided by factor
      base    the base grows by factor^(dim / (dim - 2)), which divides the slowest pair's frequency by factor and leaves the
              fastest (a head of one pair stays as it is)
      bands   pairs that turn `fast` times or more in the context stay, those that turn `slow` times or less are divided by
              factor, those between in proportion; values are scaled by 0.1 ln(factor) + 1 (published as YaRN)
    """
    if dim < 2 or dim % 2:
        raise ValueError(f"dim: {dim} values are not pairs")
    if scaling not in SCALINGS:
        raise ValueError(f"scaling {scaling!r} is none of {SCALINGS}")
    if not (base > 0 and factor > 0 and context > 0 and fast > slow > 0):
        raise ValueError("base, factor and context are positive, and fast above slow")
    j = np.arange(dim // 2, dtype=np.float64)
    if scaling == "base" and dim > 2:
        base = base * factor ** (dim / (dim - 2))
    f = base ** (-2.0 * j / dim)
    if scaling == "linear":
        return f / factor, 1.0
    if scaling != "bands":
        return f, 1.0
    keep = np.clip((context * f / (2 * math.pi) - slow) / (fast - slow), 0.0, 1.0)
    return f * (keep + (1 - keep) / factor), 0.1 * math.log(factor) + 1.0
