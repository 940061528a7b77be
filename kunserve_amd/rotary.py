"""Rotary position embedding: frequencies, part of a head, long contexts.

The reference's rotary embedding sits inside its native LlamaOp, whose source
it does not ship; the position of a step's tokens is kunserve/request.py:447-462.
"""
from __future__ import annotations

import ctypes
import math
from typing import Mapping, Optional, Sequence

import numpy as np
import torch

from . import _lib

SCALINGS = ("linear", "ntk", "yarn", "llama3")
# Keys of a scaling: those of every kind (original_max_position_embeddings has no
# part in linear and ntk), and those of one.
_KEYS = ("rope_type", "type", "factor", "rope_theta", "original_max_position_embeddings")
_KEYS_OF = dict(yarn=("beta_fast", "beta_slow", "truncate", "attention_factor", "mscale",
                      "mscale_all_dim"),
                llama3=("low_freq_factor", "high_freq_factor"))


def rotary_frequencies(rotary_dim: int, theta: float = 10000.0,
                       scaling: Optional[Mapping] = None) -> tuple:
    """(radians per position of each of rotary_dim / 2 pairs, float64; factor on
    the rotated dims).

    f_j = theta^(-2j / rotary_dim). scaling, for contexts `factor` times as long
    as those trained on, with the keys of a model configuration's rope_scaling (a
    value of None is a key left out; any other key raises, as does a rope_theta that
    is not theta):
      linear  f / factor: positions are compressed
      ntk     theta * factor^(rotary_dim / (rotary_dim - 2)): the slowest pair
              is slowed by factor, the fastest not at all
      yarn    pairs that turn more than beta_fast times within
              original_max_position_embeddings keep f, those that turn less
              than beta_slow times get f / factor, with a linear ramp over the
              pairs between, whose ends are rounded to whole pairs unless
              truncate is false; the factor on the rotated dims is
              attention_factor, by default m(mscale) / m(mscale_all_dim) where
              both are given and m(1) where neither is, m(x) = 0.1 x ln(factor) + 1
              (a softmax scale that such a model changes too is the caller's)
      llama3  the same with a ramp over the turns themselves, from
              low_freq_factor to high_freq_factor
    """
    if rotary_dim < 2 or rotary_dim % 2:
        raise ValueError(f"rotary_dim {rotary_dim} must be positive and even")
    if not (math.isfinite(theta) and theta > 0):
        raise ValueError(f"theta {theta} must be finite and positive")
    kind, factor = None, 1.0
    if scaling is not None:
        scaling = {key: x for key, x in scaling.items() if x is not None}
        kind = scaling.get("rope_type", scaling.get("type"))
        if kind != "default" and kind not in SCALINGS:
            raise ValueError(f"rope_type {kind!r} is not one of {SCALINGS}")
        if scaling.get("type", kind) != kind:
            raise ValueError(f"rope_type {kind!r} and type {scaling['type']!r} differ")
        unknown = sorted(set(scaling) - set(_KEYS) - set(_KEYS_OF.get(kind, ())))
        if unknown:
            raise ValueError(f"{kind} scaling has no {', '.join(map(repr, unknown))}")
        if float(scaling.get("rope_theta", theta)) != theta:
            raise ValueError(f"scaling has rope_theta {scaling['rope_theta']}, not {theta}")
        kind = None if kind == "default" else kind
        if kind and "factor" not in scaling:
            raise ValueError(f"{kind} scaling needs a factor")
        factor = float(scaling["factor"]) if kind else 1.0
    get = (scaling or {}).get
    if not (math.isfinite(factor) and factor >= 1):
        raise ValueError(f"scaling factor {factor} must be at least 1")
    half = rotary_dim // 2
    if kind == "ntk" and rotary_dim > 2:
        theta = theta * factor ** (rotary_dim / (rotary_dim - 2))
    f = float(theta) ** (-np.arange(half, dtype=np.float64) * (2.0 / rotary_dim))
    if kind == "linear":
        return f / factor, 1.0
    if kind not in ("yarn", "llama3"):
        return f, 1.0
    if "original_max_position_embeddings" not in scaling:
        raise ValueError(f"{kind} scaling needs original_max_position_embeddings")
    length = float(scaling["original_max_position_embeddings"])
    if not (math.isfinite(length) and length > 0):
        raise ValueError(f"original_max_position_embeddings {length} must be positive")
    if kind == "llama3":
        low, high = float(get("low_freq_factor", 1.0)), float(get("high_freq_factor", 4.0))
        if not 0 < low < high:
            raise ValueError(f"low_freq_factor {low} must be positive and below "
                             f"high_freq_factor {high}")
        keep = np.clip((f * (length / (2 * math.pi)) - low) / (high - low), 0.0, 1.0)
        return f * (keep + (1.0 - keep) / factor), 1.0
    fast, slow = float(get("beta_fast", 32.0)), float(get("beta_slow", 1.0))
    if not 0 < slow < fast:
        raise ValueError(f"beta_slow {slow} must be positive and below beta_fast {fast}")
    if theta <= 1:
        raise ValueError(f"yarn scaling needs theta above 1, got {theta}")

    def pair_of(turns):   # the (fractional) pair that turns so often within length
        return half * math.log(length / (turns * 2 * math.pi)) / math.log(theta)

    truncate = get("truncate", True)
    if truncate not in (True, False):
        raise ValueError(f"truncate {truncate!r} is neither true nor false")
    first, last = pair_of(fast), pair_of(slow)
    if truncate:
        first, last = math.floor(first), math.ceil(last)
    first, last = max(first, 0), min(last, rotary_dim - 1)
    slowed = np.clip((np.arange(half) - first) / max(last - first, 1e-3), 0.0, 1.0)
    m = [float(get(key, 1.0)) for key in ("mscale", "mscale_all_dim")]
    if ("mscale" in scaling) != ("mscale_all_dim" in scaling) or not all(0 < x < math.inf for x in m):
        raise ValueError("mscale and mscale_all_dim are positive numbers given together")
    scale = 0.1 * m[0] * math.log(factor) + 1.0
    if "mscale" in scaling:
        scale /= 0.1 * m[1] * math.log(factor) + 1.0
    scale = float(get("attention_factor", scale))
    if not math.isfinite(scale):
        raise ValueError(f"attention_factor {scale} is not finite")
    return f * (1.0 - slowed) + f / factor * slowed, scale


def _pair_axes(pairs: int, sections: Optional[Sequence[int]],
               axes: Optional[Sequence[int]]) -> Optional[np.ndarray]:
    """The axis of every pair (int32), None where there is one."""
    if sections is None and axes is None:
        return None
    if sections is not None and axes is not None:
        raise ValueError("give sections or axes")
    given = np.asarray(sections if axes is None else axes)
    if given.ndim != 1 or given.size == 0 or given.dtype.kind not in "iu" or given.min() < 0:
        raise ValueError("sections and axes are lists of whole numbers, 0 at least")
    if axes is None:
        if int(given.sum()) != pairs:
            raise ValueError(f"sections of {int(given.sum())} pairs, the rotary has {pairs}")
        return np.repeat(np.arange(given.size), given).astype(np.int32)
    if given.size != pairs:
        raise ValueError(f"the axes of {given.size} pairs, the rotary has {pairs}")
    if int(given.max()) >= 1024:
        raise ValueError("1024 axes at most")
    return given.astype(np.int32)


class Rotary:
    """Rotary embedding of the first rotary_dim dims of every head (a multiple of
    16): pairs (j, j + rotary_dim / 2), or (2j, 2j + 1) with interleave. Angles are
    formed in 64 bits, so they are exact at positions of any length.

    frequencies and scale replace those of rotary_frequencies(rotary_dim, theta,
    scaling). Use: AttentionStep.run(rope=rotary), rotary_append_kv.

    sections or axes: the tokens have a position on each of several axes (time, height
    and width of an image), and a pair turns by that on its own. sections: how many
    pairs each axis has, one axis' pairs after the other's; axes: the axis of every
    pair."""

    def __init__(self, rotary_dim: int, theta: float = 10000.0, interleave: bool = False,
                 scaling: Optional[Mapping] = None, device="cuda", frequencies=None,
                 scale: Optional[float] = None, sections: Optional[Sequence[int]] = None,
                 axes: Optional[Sequence[int]] = None):
        if rotary_dim < 16 or rotary_dim % 16:
            raise ValueError(f"rotary_dim {rotary_dim} must be a positive multiple of 16")
        if frequencies is None:
            f, factor = rotary_frequencies(rotary_dim, theta, scaling)
        else:
            if scaling is not None:
                raise ValueError("frequencies are given: scaling has no meaning")
            f, factor = np.array(frequencies, dtype=np.float64).reshape(-1), 1.0
            if f.size != rotary_dim // 2 or not np.isfinite(f).all():
                raise ValueError(f"expected {rotary_dim // 2} finite frequencies")
        self.rotary_dim = rotary_dim
        self.interleave = bool(interleave)
        self.scale = float(factor if scale is None else scale)
        if not math.isfinite(self.scale):
            raise ValueError(f"scale {self.scale} is not finite")
        pair_axis = _pair_axes(rotary_dim // 2, sections, axes)
        self.num_axes = 1 if pair_axis is None else int(pair_axis.max()) + 1
        if sections is not None:
            self.num_axes = len(sections)
        self._axes = None
        self.pair_axis = None if pair_axis is None else torch.from_numpy(pair_axis).to(device)
        self.frequencies = torch.from_numpy(f).to(device)
        self.device = self.frequencies.device
        self._desc = _lib.Rotary(self.frequencies.data_ptr(), rotary_dim, int(self.interleave),
                                 self.scale)
        self.desc = ctypes.byref(self._desc)   # as the C entries take it

    def axes_desc(self, positions: Optional[torch.Tensor]) -> Optional[_lib.RotaryAxes]:
        """The axes as the C entries take them, for positions [tokens] (one for every
        axis) or [axes, tokens]; None where there is one axis, or no positions."""
        if self.pair_axis is None or positions is None:
            return None
        stride = positions.shape[1] if positions.dim() == 2 else 0
        axes = self._axes   # the last call's serves most
        if axes is None or axes.position_stride != stride:
            self._axes = axes = _lib.RotaryAxes(self.pair_axis.data_ptr(), self.num_axes, stride)
        return axes

    def check_positions(self, positions: Optional[torch.Tensor]) -> None:
        if positions is not None and positions.dim() == 2 and positions.shape[0] != self.num_axes:
            raise ValueError(f"positions on {positions.shape[0]} axes, the rotary has "
                             f"{self.num_axes}")

    def check(self, head_dim: int, device: torch.device) -> None:
        if self.rotary_dim > head_dim:
            raise ValueError(f"rotary_dim {self.rotary_dim} exceeds head_dim {head_dim}")
        if self.device != device:
            raise ValueError(f"the rotary frequencies are on {self.device}, not {device}")
