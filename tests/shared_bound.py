"""Attention over shared prefixes in 64 bits, with the error of a kernel that takes quantized
keys as their codes."""

from __future__ import annotations

import numpy as np

from step_case import attention64, attention_bound, half_step, side64


def _sizes(fmt, pool, ids):
    """What a unit of a query is multiplied by, per token and group ``[HK, tokens, groups]``: keys
    enter as 1024 + code times the group's scale, and the bias less 1024 scales is taken
    times the queries' sum."""
    from pkv import ops

    import torch

    _, scale, bias, *_ = ops.gather_pages(fmt, pool, torch.as_tensor(ids, dtype=torch.int32, device="cuda"))
    scale, bias = (t.double().cpu().numpy() for t in (scale, bias))
    size = np.abs(scale) * (1024 + 2 ** fmt.bits - 1) + np.abs(bias - 1024 * scale)
    return size.transpose(1, 0, 2, 3).reshape(fmt.num_kv_heads, -1, size.shape[-1])


def shared64(fmt, pool, table, lens, queries, scale, *, q_pos=None, widths=None, values=None, products=None):
    """``(out, bound)`` ``[B, H, Q, D]`` over the pages' values.

    Scores: as many roundings of 2^-24 as there are ``products`` that are not zero (default D), and
    8; of quantized pages, whose keys are exact, of the terms as they enter (``_sizes``), and a bfloat16 query's conversion to float16, 2^-31 of the row's largest
    element.  Weights: float16 operands (2^-11), or two operands where results are float16
    (quantized pages) or pages bfloat16; a fixed step of 2^-31 of the largest weight in
    float16, half of it an error.  Quantized values: 2^-11 (or ``values``)."""
    import torch

    q = queries.double().cpu().numpy()
    table = table.cpu().numpy()
    batch, heads, nq, dim = q.shape
    gqa = heads // fmt.num_kv_heads
    half = half_step(torch.float16)
    f16 = fmt.quantized or fmt.dtype is torch.float16
    if fmt.quantized:
        operand = half if fmt.dtype is torch.bfloat16 else half ** 2
    else:
        operand = half if f16 else half_step(torch.bfloat16) ** 2
    value = values if values is not None else half if fmt.quantized else 0.0
    group, products = fmt.group_size, dim if products is None else products
    out, bound = np.zeros(q.shape), np.zeros(q.shape)
    for b in range(batch):
        length = int(lens[b])
        pages = -(-length // fmt.page_tokens)
        if length <= 0:
            continue
        k, v = (side64(fmt, pool, table[b, :pages], s)[:, :length] for s in (False, True))
        sizes = _sizes(fmt, pool, table[b, :pages])[:, :length] if fmt.quantized else None
        w = nq if widths is None else int(widths[b])
        for i in range(min(w, nq)):
            pos = length - w + i if q_pos is None else int(q_pos[b][i])
            sees = max(min(pos + 1, length), 0)
            if sees == 0:
                continue
            for h in range(heads):
                kh, row = h // gqa, q[b, h, i]
                o, weight, terms = attention64(row[None], k[kh], v[kh], np.array([sees]), scale)
                extra = 0.0
                if fmt.quantized:
                    by_group = np.add.reduceat(np.abs(row), np.arange(0, dim, group))
                    extra = (products + 8) * 2.0 ** -24 * float((sizes[kh, :sees] @ by_group).max())
                    if fmt.dtype is torch.bfloat16:
                        extra += dim * 2.0 ** -31 * float(np.abs(row).max() * np.abs(k[kh, :sees]).max())
                # (as ``key``, relative to the terms, and without what that adds for the values)
                key = extra / max(float(terms[0]), 1e-300)
                wide = attention_bound(o, weight, terms, scale, fmt.dtype, dim=products, tokens=length, operand=operand, key=key)
                h_out = half_step(fmt.dtype)
                wide += weight * (value - key) * (1 + h_out)
                if f16:
                    wide += length * 2.0 ** -32 * np.abs(v[kh, :sees]).max()
                out[b, h, i], bound[b, h, i] = o[0], wide[0]
    return out, bound
