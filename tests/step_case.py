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


def attention64(q, k, v, sees, scale):
    """Rows ``q [R, D]`` over ``k, v [T, D]`` (float64 arrays), row r seeing the first
    ``sees[r]`` tokens: ``(out [R, D], weight [R, D] = sum_t p_t |v_t|, terms [R] = the largest
    sum_d |q_d k_d| among the tokens seen)``.  What is not seen is not read."""
    out, weight = np.zeros(q.shape), np.zeros(q.shape)
    terms = np.zeros(len(q))
    for n in np.unique(sees):
        at = np.nonzero(sees == n)[0]
        if n <= 0:
            continue
        x = q[at] @ k[:n].T * scale
        p = np.exp(x - x.max(-1, keepdims=True))
        p /= p.sum(-1, keepdims=True)
        out[at], weight[at] = p @ v[:n], p @ np.abs(v[:n])
        terms[at] = (np.abs(q[at]) @ np.abs(k[:n]).T).max(-1)
    return out, weight, terms


def attention_bound(want, weight, terms, scale, dtype, *, dim, tokens, operand, key=0.0):
    """The error of an attention kernel's output against 64 bits.

    A score is a float32 sum of D products: at most (D + 8) roundings of 2^-24 of its terms,
    and ``key`` of them where keys enter rounded; its exponential's argument is off by as
    much times the scale (both ends of the subtraction: twice), and by 2^-22 of the range that
    is subtracted.  That moves every weight by a factor of exp(e).  Weights enter the product
    rounded by ``operand`` (their sum and their product with v: twice), values by ``key`` as
    well, and sums over the tokens are float32.  Rounding the result: half a step."""
    import torch

    eps = 2.0 ** -24
    e = 2 * abs(scale) * terms * ((dim + 8) * eps + key) + 2.0 ** -22 * (abs(scale) * terms + 16)
    rel = np.expm1(2 * e)[:, None] + 2 * operand + key + (tokens + 32) * eps
    h = half_step(dtype)
    inner = weight * rel
    return inner * (1 + h) + np.abs(want) * h + torch.finfo(dtype).smallest_normal * h
