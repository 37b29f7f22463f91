"""Tables of angles for nnc_hip_rope and nnc_hip_rope_kv_write: the cosines and
sines of position * frequency, computed in float64 (an angle of a far position
has few of float32's bits left) and rounded to float32 once."""

from __future__ import annotations

import math

import numpy as np


def frequencies(rot, base=10000.0, factor=1.0, original=None, low=1.0, high=4.0):
    """base ** (-2 i / rot) for the rot / 2 pairs, in float64.

    For contexts longer than a model was trained on, `factor` divides them: all
    of them, or, if the `original` length is given, those whose wave does not
    fit `low` times into it; a wave that fits `high` times stays, and between
    the two the share that is divided falls linearly."""
    if rot < 2 or rot % 2:
        raise ValueError(f"rot is {rot}: an even number of dims is turned")
    if not (factor > 0 and base > 0):
        raise ValueError("base and factor must be positive")
    f = float(base) ** (-np.arange(0, rot, 2, dtype=np.float64) / rot)
    if original is None:
        return f / factor
    if not high > low:
        raise ValueError("high must be larger than low")
    fits = original * f / (2 * math.pi)  # waves in the original length
    kept = np.clip((fits - low) / (high - low), 0, 1)
    return f * (kept + (1 - kept) / factor)


def angles(positions, rot, base=10000.0, amplitude=1.0, **scaling):
    """float32 [positions][rot]: rot / 2 cosines, then the sines, times `amplitude`.
    `positions`: how many, or an array of them."""
    at = np.arange(positions) if np.isscalar(positions) else np.asarray(positions)
    a = at.astype(np.float64)[:, None] * frequencies(rot, base, **scaling)
    return (amplitude * np.concatenate([np.cos(a), np.sin(a)], 1)).astype(np.float32)
