"""Rotary position embeddings in the forms that models use: pairs (i, i + dim/2)
or (2i, 2i + 1), the whole head or its first part, and angles scaled for
contexts longer than the trained one.

Pair i of a token at position p turns by p * rates[i], rates[i] =
theta^(-2i / dim), with the scaling:

  "linear"  rates / factor (positions are interpolated)
  "ntk"     theta is taken as theta * factor^(dim / (dim - 2)): the slowest
            pair is stretched by factor, the fastest not at all
  "parts"   by how often a pair turns over the trained context, n = original *
            rate / 2 pi: at alpha turns or fewer as "linear", at beta or more
            as it was, in between rate * (g + (1 - g) / factor) with
            g = (n - alpha) / (beta - alpha).  The ramp is over turns: for one
            over the pairs' numbers, or with rounded ends, take from_rates

`magnitude` multiplies the rotated values (cos and sin), for models that sharpen
attention over long contexts with it.
"""
from __future__ import annotations

import ctypes
import math

import numpy as np

from ._lib import BNR_ROPE_HALF, BNR_ROPE_INTERLEAVED, InvalidConfig, RopeDesc

__all__ = ["Rope"]


class Rope:
    """A rotation: what dev_rope and rope_scaled_table take.  ``rates``: radians
    a position of each pair (float64)."""

    LAYOUTS = {"half": BNR_ROPE_HALF, "interleaved": BNR_ROPE_INTERLEAVED}
    MAX_DIM = 512

    def __init__(self, dim: int, theta: float, layout: str = "half", scaling: str | None = None,
                 factor: float = 1.0, original: int = 0, alpha: float = 1.0, beta: float = 32.0,
                 magnitude: float = 1.0):
        if layout not in self.LAYOUTS:
            raise InvalidConfig(f"unknown rotary layout {layout!r}")
        if not isinstance(dim, int) or dim <= 0 or dim % 2 or dim > self.MAX_DIM:
            raise InvalidConfig(f"a rotary dim must be even and at most {self.MAX_DIM}, got {dim}")
        if not (math.isfinite(theta) and theta > 0):
            raise InvalidConfig(f"theta must be positive and finite, got {theta}")
        if not (math.isfinite(factor) and factor > 0):
            raise InvalidConfig(f"a scaling's factor must be positive and finite, got {factor}")
        if not math.isfinite(magnitude):
            raise InvalidConfig(f"magnitude must be finite, got {magnitude}")
        i = np.arange(dim // 2, dtype=np.float64)
        base = np.float64(theta)
        with np.errstate(all="ignore"):  # what is no number is refused below
            if scaling == "ntk":
                if dim == 2:
                    raise InvalidConfig("ntk scaling needs a rotary dim of more than 2")
                base *= np.float64(factor) ** (dim / (dim - 2))
            rates = base ** (-2.0 * i / dim)
            if scaling == "linear":
                rates = rates / factor
            elif scaling == "parts":
                if original <= 0 or not alpha < beta:
                    raise InvalidConfig("parts scaling needs original > 0 and alpha < beta, got "
                                        f"{original}, {alpha}, {beta}")
                keep = np.clip((original * rates / (2 * math.pi) - alpha) / (beta - alpha), 0, 1)
                rates = rates * (keep + (1 - keep) / factor)
            elif scaling not in (None, "ntk"):
                raise InvalidConfig(f"unknown rotary scaling {scaling!r}")
        if not (np.isfinite(base) and np.isfinite(rates).all()):
            raise InvalidConfig(f"theta {theta} with this scaling leaves rates that are no numbers")
        self._take(rates, layout, magnitude)

    @classmethod
    def from_rates(cls, rates, layout: str = "half", magnitude: float = 1.0) -> "Rope":
        """A rotation by the caller's own rates (radians a position of each pair)."""
        rates = np.array(rates, dtype=np.float64)
        if layout not in cls.LAYOUTS:
            raise InvalidConfig(f"unknown rotary layout {layout!r}")
        if rates.ndim != 1 or not 0 < 2 * rates.size <= cls.MAX_DIM or not np.isfinite(rates).all():
            raise InvalidConfig(f"rates must be 1 to {cls.MAX_DIM // 2} finite numbers")
        if not math.isfinite(magnitude):
            raise InvalidConfig(f"magnitude must be finite, got {magnitude}")
        rope = cls.__new__(cls)
        rope._take(rates, layout, magnitude)
        return rope

    def _take(self, rates, layout: str, magnitude: float) -> None:
        rates.setflags(write=False)
        self.rates, self.layout, self.magnitude, self.dim = rates, layout, float(magnitude), 2 * rates.size
        self._desc = RopeDesc(rates.ctypes.data, rates.size, self.LAYOUTS[layout], self.magnitude)
        self._ref = ctypes.byref(self._desc)
        self._fixed = True

    def __setattr__(self, name: str, value) -> None:
        # the descriptor has the rates' address
        if "_fixed" in self.__dict__:
            raise AttributeError(f"a rotation's {name} is fixed: make another one")
        object.__setattr__(self, name, value)
