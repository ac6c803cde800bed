"""Rotary positions on the GPU (not in the reference, which has no position encoding).

The first ``rotary_dim`` elements of a head are rotated in pairs by angles
``position * inv_freq[i]``: pair i is elements (i, i + rotary_dim / 2), or with
``interleaved`` (2 i, 2 i + 1).  The kernel (C ABI ``fa_apply_rotary``) computes
the angles in 64 bits, so there is no table, no largest position, and
positions far along a long context are as exact as the first ones.
"""
import math
from typing import NamedTuple, Optional

from . import _lib
from .flash_attn import _torch


class Rotary(NamedTuple):
    """A rotary position encoding: ``inv_freq`` (rotary_dim / 2,) float64 on the
    GPU, radians per position of each pair; ``interleaved`` the pairs' layout;
    ``scale`` multiplies the rotated elements (1 but for stretched contexts)."""
    inv_freq: object
    interleaved: bool = False
    scale: float = 1.0

    @property
    def rotary_dim(self) -> int:
        return 2 * self.inv_freq.shape[0]


def rotary_embedding(rotary_dim: int, base: float = 10000.0, interleaved: bool = False, scaling: Optional[str] = None,
                     factor: float = 1.0, original_length: int = 4096, beta_fast: float = 32.0, beta_slow: float = 1.0,
                     device="cuda") -> Rotary:
    """The :class:`Rotary` with frequencies ``base ** (-2 i / rotary_dim)``.
    ``scaling`` stretches the context that they were made for by ``factor``:

    * ``"linear"``: every frequency divided by ``factor``;
    * ``"ntk"``: the base raised so that the slowest pair is stretched by ``factor``
      and the fastest not at all;
    * ``"yarn"``: pairs that turn over ``beta_fast`` times within ``original_length``
      positions as they are, those under ``beta_slow`` divided by ``factor``, a ramp
      over the pairs between, and ``scale`` = 0.1 ln(factor) + 1.

    Other schemes: build the :class:`Rotary` from frequencies of your own."""
    torch = _torch()
    if rotary_dim < 2 or rotary_dim % 2:
        raise ValueError("rotary_dim must be even and positive")
    if not base > 1 or not factor >= 1:
        raise ValueError("base must be over 1 and factor at least 1")
    i = torch.arange(rotary_dim // 2, dtype=torch.float64)
    if scaling == "ntk":
        base = base * factor ** (rotary_dim / (rotary_dim - 2)) if rotary_dim > 2 else base
    freq = base ** (-2.0 * i / rotary_dim)
    scale = 1.0
    if scaling == "linear":
        freq = freq / factor
    elif scaling == "yarn":
        def pair(turns):  # where a pair turns that often within the original length
            return rotary_dim * math.log(original_length / (turns * 2 * math.pi)) / (2 * math.log(base))
        lo = max(math.floor(pair(beta_fast)), 0)
        hi = min(math.ceil(pair(beta_slow)), rotary_dim - 1)
        ramp = ((i - lo) / max(hi - lo, 0.001)).clamp(0.0, 1.0)
        freq = freq * (1 - ramp) + freq / factor * ramp
        scale = 0.1 * math.log(factor) + 1.0
    elif scaling not in (None, "ntk"):
        raise ValueError(f"unknown scaling {scaling!r}: None, 'linear', 'ntk' or 'yarn'")
    return Rotary(freq.to(device), interleaved, scale)


def _check_rotary(rotary):
    if not isinstance(rotary, Rotary):
        raise TypeError("rotary must be a Rotary (see rotary_embedding)")


def apply_rotary(query, key, rotary: Rotary, positions=None, offset: int = 0):
    """Rotates ``query`` (B, Hq, T, D) and ``key`` (B, Hkv, T, D) (or None) to
    their positions in one launch -> (query', key'), or query' alone without a key.
    Differentiable in query and key (the gradient is the rotation back; to any
    order); forward-mode derivatives are refused, and an ``inv_freq`` that
    requires grad in grad mode.

    Token t of row b is at ``positions[b, t]`` (int32 or int64, (T,) or (B, T), on the
    GPU), or at ``offset + t`` without positions.  bfloat16 or float32 with any
    strides of the first three dimensions (a projection's (B, T, H, D) output
    transposed to (B, H, T, D) is read in place); the results are dense.  Head
    dims up to 1024, any even ``rotary_dim`` up to it; multiples of 16 take 16-byte accesses, others go
    element by element (24 of 96 elements: 4.9 times the time of 32 of 96)."""
    _check_rotary(rotary)
    if positions is not None and offset:
        raise ValueError("pass positions or an offset, not both")
    return _lib.launcher().rotary(query, key, *rotary, positions, offset)
