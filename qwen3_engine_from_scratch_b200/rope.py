"""Rotary frequency plans: which angle a position each pair of a head turns by.

A plan is host arithmetic done once (in float64) and kept by the caller; the
kernels behind ``ops.rotary`` and ``ops.rotary_tables`` read it.  Unscaled, pair
i of ``rotary_dim`` elements turns by f_i = base^(-2i / rotary_dim) a position
(the reference's table, qwen3/rope.py).  For contexts longer than the
``original_len`` positions a model was trained on, by ``factor``:

``linear``  f_i / factor: every position is squeezed into the trained range.
``ntk``     the base grows to base * factor^(rotary_dim / (rotary_dim - 2)): the
            slowest pair ends at f / factor, the fastest stays.
``bands``   by the turns n_i = original_len f_i / 2 pi a pair makes over the
            trained range: at most ``slow_turns``, f_i / factor; at least
            ``fast_turns``, f_i; between, the two mixed linearly in n_i.
``yarn``    as bands, but mixed linearly in the pair's index, from the last whole
            index at which a pair makes ``fast_turns`` (or 0) to the first at which it
            makes ``slow_turns`` (at most rotary_dim - 1: the ramp may end beyond the
            last of the rotary_dim / 2 pairs).  cos and sin are scaled by
            0.1 ln(factor) + 1; a model with a factor of its own sets ``plan.gain``.

Bands and the factor on cos and sin are those of Peng et al., "YaRN: Efficient Context
Window Extension of Large Language Models", 2023, section 3; the ramp over the index is
what models that name this method are trained with.

The device form of f_i is f_i / 2 pi as a 64-bit binary fraction of a turn, from the
float64 f_i: off by up to 2^-54 turns a position.
"""

from __future__ import annotations

import math

import torch

LAYOUTS = ("half", "interleaved")
SCALINGS = (None, "linear", "ntk", "bands", "yarn")


def rotary_frequencies(rotary_dim, base=10000.0, scaling=None, factor=1.0, original_len=None,
                       slow_turns=1.0, fast_turns=32.0):
    """(float64 list of rotary_dim / 2 angles a position, gain on cos and sin)."""
    if rotary_dim < 2 or rotary_dim % 2:
        raise ValueError(f"rotary_dim must be even and at least 2 (got {rotary_dim})")
    if not base > 1.0 or not math.isfinite(base):
        raise ValueError(f"base must be finite and above 1 (got {base})")
    if scaling not in SCALINGS:
        raise ValueError(f"scaling must be one of {SCALINGS} (got {scaling!r})")
    if scaling is not None and not (factor >= 1.0 and math.isfinite(factor)):
        raise ValueError(f"factor must be finite and at least 1 (got {factor})")
    half = rotary_dim // 2
    if scaling == "ntk":
        if rotary_dim == 2:
            raise ValueError("ntk scaling needs rotary_dim of at least 4")
        base = base * factor ** (rotary_dim / (rotary_dim - 2))
    freq = [base ** (-2.0 * i / rotary_dim) for i in range(half)]
    if scaling is None or scaling == "ntk":
        return freq, 1.0
    if scaling == "linear":
        return [f / factor for f in freq], 1.0
    if original_len is None or original_len < 1:
        raise ValueError(f"{scaling} scaling needs original_len")
    if not 0 < slow_turns < fast_turns:
        raise ValueError("0 < slow_turns < fast_turns is needed")
    if scaling == "bands":
        keep = [(original_len * f / (2 * math.pi) - slow_turns) / (fast_turns - slow_turns)
                for f in freq]
        gain = 1.0
    else:
        def index(turns):   # where original_len * base^(-2i / rotary_dim) = 2 pi turns
            return rotary_dim * math.log(original_len / (2 * math.pi * turns)) / (2 * math.log(base))

        first = max(math.floor(index(fast_turns)), 0)
        last = min(math.ceil(index(slow_turns)), rotary_dim - 1)
        keep = [1.0 - (i - first) / max(last - first, 1e-3) for i in range(half)]
        gain = 0.1 * math.log(factor) + 1.0
    keep = [min(1.0, max(0.0, k)) for k in keep]
    return [f * (k + (1.0 - k) / factor) for f, k in zip(freq, keep)], gain


class RotaryPlan:
    """Frequencies of ``rotary_dim`` elements on ``device``, for ``ops.rotary``
    and ``ops.rotary_tables``.  ``layout``: "half" pairs element i with
    i + rotary_dim / 2, "interleaved" 2i with 2i + 1."""

    def __init__(self, rotary_dim, base=10000.0, layout="half", scaling=None, factor=1.0,
                 original_len=None, slow_turns=1.0, fast_turns=32.0, device="cuda"):
        if layout not in LAYOUTS:
            raise ValueError(f"layout must be one of {LAYOUTS} (got {layout!r})")
        self.rotary_dim, self.layout = int(rotary_dim), layout
        self.interleaved = layout == "interleaved"
        self.freq, self.gain = rotary_frequencies(self.rotary_dim, base, scaling, factor,
                                                  original_len, slow_turns, fast_turns)
        self.turns = torch.tensor([_signed64(round(f / (2 * math.pi) * 2.0 ** 64)) for f in self.freq],
                                  dtype=torch.int64, device=device)


def _signed64(v):
    v &= (1 << 64) - 1
    return v - (1 << 64) if v >> 63 else v
