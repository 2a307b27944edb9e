"""Shared helpers of the tests of a serving step's operators: projections, pages and
results in 64 bits."""

from __future__ import annotations

import numpy as np


def half_step(dtype):
    """The most that rounding to ``dtype`` moves a value, relative to it."""
    import torch

    return torch.finfo(dtype).eps / 2


def turned64(x, angles, half):
    """Heads ``x [..., heads, D]`` (float64) with pairs (i, i + half) turned by ``angles
    [..., half]``, and the sizes of the terms each element is a sum of."""
    cos, sin = np.cos(angles)[..., None, :], np.sin(angles)[..., None, :]
    a, b = x[..., :half], x[..., half:2 * half]
    y, size = x.copy(), np.zeros_like(x)
    y[..., :half], y[..., half:2 * half] = a * cos - b * sin, b * cos + a * sin
    size[..., :half] = size[..., half:2 * half] = np.abs(a) + np.abs(b)
    return y, size


def assert_turned(got, want, size, dtype):
    """``got`` (of ``dtype``) within its rounding of ``want``: half a step, and before it
    cos or sin rounded to 32 bits, two products and a sum: 4 roundings of 2^-24 of the
    terms (and what rounding does to that)."""
    import torch

    got = got.double().cpu().numpy()
    h = half_step(dtype)
    bound = np.abs(want) * h + 4 * 2.0 ** -24 * size * (1 + h) + torch.finfo(dtype).smallest_normal * h
    off = np.abs(got - want)
    assert np.all(off <= bound), float(np.nanmax(off / bound))
