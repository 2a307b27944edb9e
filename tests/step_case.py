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


def side64(fmt, pool, ids, values):
    """K or V of pages ``ids`` as ``[HK, pages * page_tokens, D]`` float64."""
    import torch

    from cache_ops_case import _dequantized
    from pkv import ops

    ids = torch.as_tensor(ids, dtype=torch.int32, device="cuda")
    parts = ops.gather_pages(fmt, pool, ids)
    if fmt.quantized:
        x, _ = _dequantized(*(parts[3:] if values else parts[:3]), fmt.bits, fmt.group_size, fmt.head_dim)
    else:
        x = parts[int(values)].double().cpu().numpy()
    return x.transpose(1, 0, 2, 3).reshape(fmt.num_kv_heads, -1, fmt.head_dim)


def paged64(fmt, pool, table, lens, queries, scale, *, q_pos=None, widths=None):
    """``(out, bound)`` ``[B, H, Q, D]``: paged attention in 64 bits over the pages' values, and
    the error of a kernel whose keys, values and weights of quantized pages are rounded to
    float16 operands (of float pages: the keys and values as they are, bfloat16 weights to
    twice their bits)."""
    import torch

    q = queries.double().cpu().numpy()
    table = table.cpu().numpy()
    batch, heads, nq, dim = q.shape
    gqa = heads // fmt.num_kv_heads
    half = half_step(torch.float16)
    key = half if fmt.quantized else 0.0
    operand = half if fmt.quantized or fmt.dtype is torch.float16 else half_step(torch.bfloat16) ** 2
    out, bound = np.zeros(q.shape), np.zeros(q.shape)
    for b in range(batch):
        length = min(int(lens[b]), table.shape[1] * fmt.page_tokens)
        pages = -(-max(length, 0) // fmt.page_tokens)
        mapped = (table[b, :pages] >= 0) & (table[b, :pages] < pool.shape[0])
        if length <= 0 or not mapped.any():
            continue
        ids = np.where(mapped, table[b, :pages], 0)
        there = np.repeat(mapped, fmt.page_tokens)[:length]
        k, v = (side64(fmt, pool, ids, s)[:, :length][:, there] for s in (False, True))
        w = nq if widths is None else int(widths[b])
        for i in range(min(w, nq)):
            pos = int(lens[b]) - w + i if q_pos is None else int(q_pos[b][i])
            sees = int(there[:max(min(pos + 1, length), 0)].sum())
            for h in range(heads):
                with np.errstate(invalid="ignore", over="ignore"):
                    o, weight, terms = attention64(q[b, h, i:i + 1], k[h // gqa], v[h // gqa], np.array([sees]), scale)
                out[b, h, i] = o[0]
                bound[b, h, i] = attention_bound(o, weight, terms, scale, fmt.dtype, dim=dim, tokens=length,
                                                 operand=operand, key=key)[0]
    return out, bound
