"""Rotary tables: the cosines and sines that ``ops.rotary`` and
``ops.append_tokens`` read, built once per model.

A table is fp32 ``[max_pos, dim]``: row p holds cos(p f_i) for the dim/2 pairs,
then sin(p f_i), with f_i = theta^(-2i/dim), or stretched for contexts longer
than the trained one (:class:`RopeScaling`).  Angles are formed in float64 (a
far position times a frequency has no useful float32 value) and rounded once.
Both pair layouts (half and interleaved) read the same table.
Reference: rope.py:25-84 build_rope_cache.
"""

from __future__ import annotations

import math
from dataclasses import dataclass

import torch


@dataclass(frozen=True)
class RopeScaling:
    """How a table reaches ``factor`` times the trained context.

    * ``linear``: positions divided by the factor.
    * ``ntk``: theta raised to theta * factor^(dim / (dim - 2)), which leaves the
      fastest pair as it is and slows the slowest by the factor.
    * ``yarn``: pairs that turn more than ``beta_fast`` times within
      ``original_max_pos`` stay, those below ``beta_slow`` turns are slowed by the
      factor, with a linear ramp over the pairs between; the table is
      multiplied by (0.1 mscale ln(factor) + 1) / (0.1 mscale_all_dim ln(factor)
      + 1) (YaRN, Peng et al. 2023; the quotient's second term is for models
      that put it into the softmax scale).
    """

    kind: str
    factor: float
    original_max_pos: int = 4096
    beta_fast: float = 32.0
    beta_slow: float = 1.0
    mscale: float = 1.0
    mscale_all_dim: float = 0.0

    def __post_init__(self) -> None:
        if self.kind not in ("linear", "ntk", "yarn"):
            raise ValueError(f"unknown rope scaling '{self.kind}'; choose linear, ntk or yarn")
        if not self.factor >= 1.0 or math.isinf(self.factor):
            raise ValueError(f"the factor must be finite and at least 1, got {self.factor}")
        if self.original_max_pos < 1 or not 0 < self.beta_slow <= self.beta_fast:
            raise ValueError("original_max_pos must be >= 1 and 0 < beta_slow <= beta_fast")


def rope_frequencies(dim: int, theta: float = 10000.0, scaling: RopeScaling | None = None) -> torch.Tensor:
    """Angle per position of the dim/2 pairs, float64 on the CPU."""
    if dim < 2 or dim % 2:
        raise ValueError(f"the rotated part must be a positive even number of values, got {dim}")
    if not theta > 1.0:
        raise ValueError(f"theta must be above 1, got {theta}")
    if scaling is not None and scaling.kind == "ntk":
        if dim == 2:
            raise ValueError("ntk scaling needs at least two pairs")
        theta = theta * scaling.factor ** (dim / (dim - 2))
    i = torch.arange(dim // 2, dtype=torch.float64)
    f = theta ** (-2.0 * i / dim)
    if scaling is None or scaling.kind == "ntk":
        return f
    if scaling.kind == "linear":
        return f / scaling.factor

    def pair_of(turns: float) -> float:  # the pair that turns so often within the trained context
        return dim * math.log(scaling.original_max_pos / (2 * math.pi * turns)) / (2 * math.log(theta))
    lo = max(math.floor(pair_of(scaling.beta_fast)), 0)
    hi = min(math.ceil(pair_of(scaling.beta_slow)), dim - 1)
    if hi <= 0:  # not even the first pair turns beta_slow times
        return f / scaling.factor
    ramp = ((i - lo) / max(hi - lo, 1e-3)).clamp(0.0, 1.0)
    return f * (1.0 - ramp) + f / scaling.factor * ramp


def build_rope_table(max_pos: int, dim: int = 64, theta: float = 10000.0, scaling: RopeScaling | None = None,
                     device=None) -> torch.Tensor:
    """[max_pos, dim] fp32: the cosines of the dim/2 pairs, then their sines."""
    if max_pos < 1:
        raise ValueError(f"max_pos must be >= 1, got {max_pos}")
    f = rope_frequencies(dim, theta, scaling).to(device)
    angle = torch.arange(max_pos, dtype=torch.float64, device=f.device)[:, None] * f
    m = 1.0
    if scaling is not None and scaling.kind == "yarn":
        ln = 0.1 * math.log(scaling.factor)
        m = (scaling.mscale * ln + 1.0) / (scaling.mscale_all_dim * ln + 1.0)
    return torch.cat([angle.cos() * m, angle.sin() * m], dim=1).float().contiguous()
