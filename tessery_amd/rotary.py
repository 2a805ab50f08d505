"""Frequencies and tables of rotary positions (HipRuntime._rotary), for trained and longer contexts.

Pair c of a head's `dim` rotated channels turns by theta^(-2c / dim) radians a position. For contexts
`factor` times as long as the model was trained on:
  linear  every frequency divided by the factor (positions squeezed into the trained range)
  ntk     theta raised so that the slowest pair is divided by the factor and the fastest kept:
          theta * factor^(dim / (dim - 2))
  yarn    pairs that make at least `fast` turns within the trained length are kept, those of at most
          `slow` turns divided by the factor, and those between blended linearly in their turns; the
          rotated channels are multiplied by 0.1 ln(factor) + 1
Other schemes: make the float64 frequencies and pass them to table().
"""

from __future__ import annotations

import math
from typing import TYPE_CHECKING

import numpy as np
from numpy.typing import NDArray

from .errors import InferenceError

if TYPE_CHECKING:
    from .runtime import Buffer, HipRuntime

SCALINGS = ("none", "linear", "ntk", "yarn")


def frequencies(dim: int, theta: float, *, scaling: str = "none", factor: float = 1.0,
                trained: int = 0, slow: float = 1.0,
                fast: float = 32.0) -> tuple[NDArray[np.float64], float]:
    """Radians a position of each of the dim / 2 pairs, and the factor on the rotated channels.
    `trained`: the length the unscaled frequencies were trained for (yarn)."""
    if type(dim) is not int or dim < 2 or dim % 2 or not 0.0 < theta < math.inf or \
            scaling not in SCALINGS or not 1.0 <= factor < math.inf:
        raise InferenceError()
    pairs = np.arange(dim // 2, dtype=np.float64)
    if scaling == "ntk" and dim > 2:
        theta = theta * factor ** (dim / (dim - 2))
    base = theta ** (-2.0 * pairs / dim)
    if scaling == "linear":
        return base / factor, 1.0
    if scaling == "yarn":
        if trained < 1 or not 0.0 <= slow < fast:
            raise InferenceError()
        turns = trained * base / (2.0 * math.pi)
        kept = np.clip((turns - slow) / (fast - slow), 0.0, 1.0)
        return base * kept + base / factor * (1.0 - kept), 0.1 * math.log(factor) + 1.0
    return base, 1.0


def table(runtime: HipRuntime, *, positions: int, dim: int, theta: float = 1e6,
          scaling: str = "none", factor: float = 1.0, trained: int = 0,
          values: NDArray[np.float64] | None = None, multiplier: float = 1.0) -> Buffer:
    """The buffer _rotary reads, for positions 0 .. positions - 1: the frequencies of frequencies(),
    or `values` (float64 [dim / 2]) with `multiplier` on the rotated channels. Made in a command of
    its own and kept like a weight."""
    if values is None:
        values, multiplier = frequencies(dim, theta, scaling=scaling, factor=factor,
                                         trained=trained)
    values = np.ascontiguousarray(values, np.float64)
    if type(positions) is not int or positions < 1 or values.shape != (dim // 2,) or \
            not np.isfinite(values).all():
        raise InferenceError()
    source = runtime.upload(values)
    made = None
    try:
        made = runtime.buffer(positions * dim * 4)
        with runtime.command():
            runtime._rotary_table([source, made], positions=positions, rotary_dim=dim,
                                  factor=multiplier)
        return made
    except BaseException:
        if made is not None:
            made.close()
        raise
    finally:
        source.close()
