"""Angles of rotary positions: how far each pair of a head's values turns a position.

A pair i of ``size`` rotated values turns by ``base ** (-2 i / size)`` radians a position, changed for long
contexts by a scaling:

  linear  all of them by 1 / factor
  ntk     base * factor ** (size / (size - 2)) in the place of base
  llama3  those of a wavelength above original_length / low_freq_factor by 1 / factor, those below
          original_length / high_freq_factor not at all, between them in proportion
  yarn    by 1 / factor where a pair turns fewer than beta_slow times over original_length, not at all
          where it turns more than beta_fast times, between them in proportion to i; rotated values are
          multiplied by ``magnitude`` (0.1 ln(factor) + 1 unless it is given)

The kernels take the angles as fractions of a turn in 64 bits, whose product with a position wraps where the
angle does: positions lose no precision however far they are. The reference has no counterpart.
"""

from __future__ import annotations

import math
from dataclasses import dataclass
from typing import Sequence

import torch

from mambo_amd import _native

MAX_ROTARY_DIM = 1024  # MAMBO_ROTARY_MAX_DIM

_NEEDED = {"linear": {"factor"}, "ntk": {"factor"},
           "llama3": {"factor", "low_freq_factor", "high_freq_factor", "original_length"},
           "yarn": {"factor", "original_length"}}
_OPTIONAL = {"yarn": {"beta_fast", "beta_slow", "magnitude"}}


@dataclass(frozen=True)
class RotaryTable:
    """Prepared angles: ``turns`` int64 [size / 2] (the bits of unsigned fractions of a turn times 2^64),
    ``size`` rotated values a head, in pairs of neighbours (``interleaved``) or (i, i + size / 2), and the
    ``magnitude`` that multiplies them."""

    turns: torch.Tensor
    size: int
    interleaved: bool
    magnitude: float

    def __post_init__(self):
        if self.size < 2 or self.size % 2 or tuple(self.turns.shape) != (self.size // 2,) or self.turns.dtype != torch.int64 \
                or not self.turns.is_contiguous():
            raise ValueError(f"angles of {self.size} values are contiguous int64 [{self.size // 2}]")
        object.__setattr__(self, "args", _native.RotaryTableArgs(self.turns.data_ptr(), self.size, self.interleaved,
                                                                 self.magnitude))

    def __reduce__(self):  # a copy's tensor is its own, and so is the address that it hands to the kernels
        return RotaryTable, (self.turns, self.size, self.interleaved, self.magnitude)


def rotary_frequencies(size: int, *, base: float = 10000.0, scaling: dict | None = None) -> tuple[list[float], float]:
    """Radians a position of each of the size / 2 pairs, and the magnitude, in Python's 64-bit floats."""
    if not isinstance(size, int) or isinstance(size, bool) or size < 2 or size % 2 or size > MAX_ROTARY_DIM:
        raise ValueError(f"an even number of values is rotated, up to {MAX_ROTARY_DIM} (got {size})")
    if not (math.isfinite(base) and base > 1.0):
        raise ValueError(f"base must be finite and above 1 (got {base})")
    if scaling is None:
        return [base ** (-2.0 * i / size) for i in range(size // 2)], 1.0
    kind = scaling.get("type")
    given = {k: float(v) for k, v in scaling.items() if k != "type"}
    if kind not in _NEEDED:
        raise ValueError(f"scaling type must be one of {sorted(_NEEDED)} (got {kind!r})")
    missing, unknown = _NEEDED[kind] - set(given), set(given) - _NEEDED[kind] - _OPTIONAL.get(kind, set())
    if missing or unknown:
        raise ValueError(f"scaling {kind}: missing {sorted(missing)}, unknown {sorted(unknown)}")
    if not all(math.isfinite(v) and v > 0.0 for v in given.values()):
        raise ValueError("scaling values must be finite and positive")
    factor = given["factor"]
    if kind == "ntk":
        if size == 2:
            raise ValueError("ntk scaling needs more than one pair")
        base = base * factor ** (size / (size - 2.0))
    plain = [base ** (-2.0 * i / size) for i in range(size // 2)]
    if kind == "ntk":
        return plain, 1.0
    if kind == "linear":
        return [f / factor for f in plain], 1.0
    if kind == "llama3":
        low, high, length = given["low_freq_factor"], given["high_freq_factor"], given["original_length"]
        if high <= low:
            raise ValueError("high_freq_factor must be above low_freq_factor")
        keep = [min(1.0, max(0.0, (length * f / (2.0 * math.pi) - low) / (high - low))) for f in plain]
        return [f * (k + (1.0 - k) / factor) for f, k in zip(plain, keep)], 1.0
    fast, slow, length = given.get("beta_fast", 32.0), given.get("beta_slow", 1.0), given["original_length"]
    if fast <= slow:
        raise ValueError("beta_fast must be above beta_slow")

    def pair_of(turns: float) -> float:  # the pair that turns so many times over the original length
        return size * math.log(length / (2.0 * math.pi * turns)) / (2.0 * math.log(base))

    low, high = max(math.floor(pair_of(fast)), 0), min(math.ceil(pair_of(slow)), size - 1)
    ramp = [min(1.0, max(0.0, (i - low) / max(high - low, 0.001))) for i in range(size // 2)]
    return ([f * (1.0 - r + r / factor) for f, r in zip(plain, ramp)],
            given.get("magnitude", 0.1 * math.log(factor) + 1.0 if factor > 1.0 else 1.0))


def prepare_rotary_table(size: int, *, base: float = 10000.0, scaling: dict | None = None, interleaved: bool = False,
                         frequencies: Sequence[float] | None = None, device=None) -> RotaryTable:
    """The angles of ``size`` rotated values a head on a GPU (default: the current one), by ``base`` and
    ``scaling`` (a dict of ``type`` and its values), or by ``frequencies``, radians a position of each
    pair, of any other scheme."""
    if frequencies is None:
        radians, magnitude = rotary_frequencies(size, base=base, scaling=scaling)
    else:
        rotary_frequencies(size)
        radians, magnitude = [float(f) for f in frequencies], 1.0
        if scaling is not None or len(radians) != size // 2 or not all(math.isfinite(f) for f in radians):
            raise ValueError(f"frequencies must be {size // 2} finite values, without a scaling")
    bits = []
    for f in radians:
        turn = math.fmod(f / (2.0 * math.pi), 1.0)
        word = round(turn * 2.0**64) % 2**64
        bits.append(word - 2**64 if word >= 2**63 else word)
    device = torch.device("cuda", torch.cuda.current_device()) if device is None else torch.device(device)
    if device.type != "cuda":
        raise ValueError("the angles must be on a GPU")
    return RotaryTable(torch.tensor(bits, dtype=torch.int64, device=device), size, bool(interleaved), float(magnitude))
