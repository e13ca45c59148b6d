"""The cos / sin tables that the rotary kernels read, formed in 64 bits and rounded once to f32.

An angle is position * frequency: at position 10^6 a frequency's f32 rounding (2^-24 relative)
moves the angle by 0.06 radians, so positions and frequencies stay in float64 until the cosine.
A program makes the tables once, for the longest context it serves, and keeps them in device
memory next to its weights.

Contexts longer than the frequencies were made for:

* ``linear``: positions divided by ``factor``;
* ``ntk``: the base raised to base * factor^(R / (R - 2)), which leaves the fastest pair as it is
  and slows the slowest by ``factor``;
* ``parts``: with r = original * frequency / (2 pi) the turns that a pair makes over the original
  context, its frequency is kept where r > ``fast``, divided by ``factor`` where r < ``slow``, and in
  between f ((1 - g) / factor + g), g = (r - slow) / (fast - slow); cos and sin are then scaled by
  ``scale`` (Peng et al., "YaRN: Efficient Context Window Extension of Large Language Models", 2023,
  whose own choice for the scale is 0.1 ln(factor) + 1).
"""

from __future__ import annotations

import math

import numpy as np

SCALINGS = (None, "linear", "ntk", "parts")


def frequencies(rotary: int, base: float = 10000.0, scaling: str | None = None, factor: float = 1.0,
                original: int | None = None, fast: float = 32.0, slow: float = 1.0) -> np.ndarray:
    """float64 [rotary / 2]: radians per position of each pair."""
    if rotary < 2 or rotary % 2:
        raise ValueError(f"rotary = {rotary}: an even number of at least 2 expected")
    if scaling not in SCALINGS:
        raise ValueError(f"scaling {scaling!r} (one of {', '.join(map(str, SCALINGS))})")
    if not base > 0 or not factor >= 1:
        raise ValueError(f"base {base!r} and factor {factor!r}: base > 0 and factor >= 1 expected")
    i = np.arange(rotary // 2, dtype=np.float64)
    if scaling == "ntk" and rotary > 2:
        base = base * factor ** (rotary / (rotary - 2))
    f = float(base) ** (-2.0 * i / rotary)
    if scaling == "linear":
        return f / factor
    if scaling == "parts":
        if not original or original < 1:
            raise ValueError("parts scaling needs the original context length")
        if not fast > slow > 0:
            raise ValueError(f"parts scaling: fast {fast!r} > slow {slow!r} > 0 expected")
        g = np.clip((original * f / (2 * math.pi) - slow) / (fast - slow), 0.0, 1.0)
        return f * ((1 - g) / factor + g)
    return f


def tables(rows: int, rotary: int, base: float = 10000.0, scaling: str | None = None, factor: float = 1.0,
           original: int | None = None, fast: float = 32.0, slow: float = 1.0,
           scale: float = 1.0) -> tuple[np.ndarray, np.ndarray]:
    """(cos, sin), f32 [rows, rotary / 2]: row p holds ``scale`` times cos and sin of position p's
    angles."""
    if rows < 1:
        raise ValueError(f"rows = {rows}: a positive number expected")
    f = frequencies(rotary, base, scaling, factor, original, fast, slow)
    cos = np.empty((rows, rotary // 2), dtype=np.float32)
    sin = np.empty_like(cos)
    for p0 in range(0, rows, 65536):                  # bounds the float64 temporaries
        a = np.arange(p0, min(rows, p0 + 65536), dtype=np.float64)[:, None] * f
        cos[p0:p0 + len(a)] = np.cos(a) * scale
        sin[p0:p0 + len(a)] = np.sin(a) * scale
    return cos, sin
