"""Angle tables of rotary positions (``kernels.rope`` applies them).

A channel pair m of an axis with d channels turns by ``position * f_m`` with
``f_m = theta ** (-2m / d)``; a token of a video grid has one position per
axis (t, h, w), whose channels follow each other in the head.  Angles are
formed in 64 bits (in 32 bits position 100000 is off by several thousandths
of a radian on the fastest pair) and stored as fp32 cos and sin, once per
geometry.

Longer contexts than the model was trained on (``RopeScaling``):

* ``linear``: every position divided by ``factor``;
* ``ntk``: ``theta * factor ** (d / (d - 2))``, which stretches the slowest
  pair by ``factor`` and leaves the fastest alone;
* ``yarn``: pair by pair, with r = trained length / wavelength: divided by
  ``factor`` for r < ``low``, untouched for r > ``high``, mixed linearly in
  between; cos and sin times ``0.1 ln(factor) + 1``.
"""
from __future__ import annotations

import math
from dataclasses import dataclass
from typing import Optional, Sequence, Tuple

import torch

from .geometry import VideoGeometry


@dataclass(frozen=True)
class RopeScaling:
    kind: str                     # "linear", "ntk" or "yarn"
    factor: float                 # how many times longer than trained (>= 1)
    trained_len: Optional[int] = None  # positions per axis the model saw; yarn needs it
    low: float = 1.0
    high: float = 32.0

    def __post_init__(self):
        if self.kind not in ("linear", "ntk", "yarn"):
            raise ValueError(f"scaling kind must be linear, ntk or yarn, got {self.kind!r}")
        if not self.factor >= 1.0 or math.isinf(self.factor):
            raise ValueError(f"scaling factor must be at least 1, got {self.factor}")
        if self.kind == "yarn" and (self.trained_len is None or self.trained_len < 1):
            raise ValueError("yarn scaling needs trained_len")
        if self.low >= self.high:
            raise ValueError(f"low {self.low} must be below high {self.high}")


@dataclass(frozen=True)
class RopeTable:
    """fp32 ``[tokens, R/2]`` cos and sin of the tokens after the first
    ``text_len``, and the pair layout they are meant for."""

    cos: torch.Tensor
    sin: torch.Tensor
    text_len: int = 0
    layout: str = "interleaved"


def rope_freqs(dim: int, theta: float = 10000.0, scaling: Optional[RopeScaling] = None,
               device="cpu") -> torch.Tensor:
    """fp64 ``[dim / 2]`` angles per unit of position of one axis."""
    if dim < 0 or dim % 2:
        raise ValueError(f"an axis takes an even number of channels, got {dim}")
    if not theta > 0:
        raise ValueError(f"theta must be positive, got {theta}")
    if scaling is not None and scaling.kind == "ntk" and dim > 2:
        theta = theta * scaling.factor ** (dim / (dim - 2))
    f = theta ** (-torch.arange(0, dim, 2, dtype=torch.float64, device=device) / max(dim, 1))
    if scaling is None or scaling.kind == "ntk":
        return f
    if scaling.kind == "linear":
        return f / scaling.factor
    turns = scaling.trained_len * f / (2.0 * math.pi)
    keep = ((turns - scaling.low) / (scaling.high - scaling.low)).clamp(0.0, 1.0)
    return f * (keep + (1.0 - keep) / scaling.factor)


def rope_table(positions: torch.Tensor, dims: Sequence[int], theta: float = 10000.0,
               scaling: Optional[RopeScaling] = None) -> Tuple[torch.Tensor, torch.Tensor]:
    """fp32 cos and sin ``[..., sum(dims) / 2]`` of ``positions`` ``[...,
    len(dims)]`` (any number type, on the device that the tables shall have)."""
    if positions.dim() < 1 or positions.shape[-1] != len(dims):
        raise ValueError(f"positions {tuple(positions.shape)} need one value for each of {len(dims)} axes")
    pos = positions.to(torch.float64)
    angle = torch.cat([pos[..., i:i + 1] * rope_freqs(d, theta, scaling, pos.device) for i, d in enumerate(dims)],
                      dim=-1)
    amp = 0.1 * math.log(scaling.factor) + 1.0 if scaling is not None and scaling.kind == "yarn" else 1.0
    return (angle.cos() * amp).float(), (angle.sin() * amp).float()


def video_rope(geo: VideoGeometry, head_dim: int = 64, dims: Optional[Sequence[int]] = None, *,
               theta: float = 10000.0, layout: str = "interleaved", scaling: Optional[RopeScaling] = None,
               device="cpu") -> RopeTable:
    """Table of the video tokens of ``geo`` (text first, unrotated), positions
    = their (t, h, w) grid indexes.  ``dims``: channels of the three axes, by
    default the whole head as 2 : 3 : 3 (16, 24, 24 of 64)."""
    if dims is None:
        if head_dim % 16:
            raise ValueError(f"head_dim {head_dim} does not split 2 : 3 : 3 into even parts; pass dims")
        dims = (head_dim // 4, head_dim // 8 * 3, head_dim // 8 * 3)
    if sum(dims) > head_dim or sum(dims) == 0:
        raise ValueError(f"axes {tuple(dims)} do not fit into {head_dim} channels")
    t, h, w = (torch.arange(n, device=device) for n in (geo.frames, geo.height, geo.width))
    grid = torch.stack(torch.meshgrid(t, h, w, indexing="ij"), dim=-1).reshape(geo.video_len, 3)
    cos, sin = rope_table(grid, dims, theta, scaling)
    return RopeTable(cos, sin, geo.text_len, layout)
