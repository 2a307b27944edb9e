"""Shared helpers of the tests of attention mass, eviction, beams and reordering:
pages filled through the library, and their contents in 64 bits."""

from __future__ import annotations

import math

import numpy as np


def filled(fmt, lens, *, seed=0, extra_pages=0, junk=0xFF, k_scale=1.0):
    """A pool whose every byte is ``junk`` but for the appended tokens of sequences of
    ``lens`` tokens, on shuffled pages; ``(pool, table [B, most + 1], spare page ids)``."""
    import torch

    from pkv import ops

    rng = np.random.default_rng(seed)
    p = fmt.page_tokens
    counts = [-(-n // p) for n in lens]
    total = sum(counts) + extra_pages
    ids = rng.permutation(max(total, 1)).astype(np.int32)
    table = np.full((len(lens), max(counts, default=0) + 1), -1, np.int32)
    at = 0
    for b, n in enumerate(counts):
        table[b, :n] = ids[at:at + n]
        at += n
    pool = ops.allocate_pool(fmt, max(total, 1))
    pool.fill_(junk)
    longest = max(max(lens, default=1), 1)
    shape = (len(lens), fmt.num_kv_heads, longest, fmt.head_dim)
    k = torch.from_numpy(rng.standard_normal(shape).astype(np.float32) * k_scale).cuda().to(fmt.dtype)
    v = torch.from_numpy(rng.standard_normal(shape).astype(np.float32)).cuda().to(fmt.dtype)
    table = torch.from_numpy(table).cuda()
    width = torch.tensor(lens, dtype=torch.int32, device="cuda")
    ops.append_quantize(fmt, pool, k, v, table, torch.zeros_like(width), width)
    return pool, table, ids[at:]


def _dequantized(codes, scale, bias, bits, group, dim):
    codes = codes.cpu().numpy()
    if bits == 4:
        codes = np.stack((codes & 15, codes >> 4), -1).reshape(*codes.shape[:-1], -1)
    s, b = (np.repeat(x.cpu().numpy().astype(np.float64), group, -1) for x in (scale, bias))
    return (codes * s + b)[..., :dim], (codes * np.abs(s) + np.abs(b))[..., :dim]


def keys64(fmt, pool, ids):
    """K of pages ``ids`` as ``[HK, pages * page_tokens, D]`` float64, and the sizes of
    the terms each element is a sum of."""
    import torch

    from pkv import ops

    ids = torch.as_tensor(ids, dtype=torch.int32, device="cuda")
    parts = ops.gather_pages(fmt, pool, ids)
    if fmt.quantized:
        k, size = _dequantized(*parts[:3], fmt.bits, fmt.group_size, fmt.head_dim)
    else:
        k = parts[0].double().cpu().numpy()
        size = np.abs(k)
    return tuple(x.transpose(1, 0, 2, 3).reshape(fmt.num_kv_heads, -1, fmt.head_dim) for x in (k, size))


def mass64(fmt, pool, table, lens, queries, scale, *, q_pos=None, widths=None):
    """``[B] of [HK, T]`` attention weight per token in float64, and a bound of the
    error of the same in float32.

    A score is a float32 sum of D products, of the group offsets and of a product
    with the scale: at most (D + 16) roundings of 2^-24 of the sum of the terms'
    sizes, e in all; each weight is then off by a factor of at most exp(2 e), by the
    roundings of its exponential (argument reduced and scaled: 8 steps and |s| 2^-22)
    and of the sums over the tokens and over the rows (one per term)."""
    q = queries.double().cpu().numpy()
    table = table.cpu().numpy()
    batch, heads, nq, dim = q.shape
    gqa = heads // fmt.num_kv_heads
    eps = 2.0 ** -24
    out, bound = [], []
    for b in range(batch):
        length = min(int(lens[b]), table.shape[1] * fmt.page_tokens)
        total, err = (np.zeros((fmt.num_kv_heads, max(length, 0))) for _ in range(2))
        pages = -(-max(length, 0) // fmt.page_tokens)
        mapped = (table[b, :pages] >= 0) & (table[b, :pages] < pool.shape[0])
        if length > 0 and mapped.any():
            k, size = keys64(fmt, pool, np.where(mapped, table[b, :pages], 0))
            k, size = k[:, :length], size[:, :length]
            there = np.repeat(mapped, fmt.page_tokens)[:length]
            w = nq if widths is None else int(widths[b])
            for i in range(min(w, nq)):
                pos = int(lens[b]) - w + i if q_pos is None else int(q_pos[b][i])
                see = there & (np.arange(length) <= pos)
                if not see.any():
                    continue
                rows = q[b, :, i].reshape(fmt.num_kv_heads, gqa, dim)
                s = np.einsum("hgd,htd->hgt", rows, np.where(there[None, :, None], k, 0)) * scale
                terms = np.einsum("hgd,htd->hgt", np.abs(rows), np.where(there[None, :, None], size, 0))
                e = (dim + 16) * eps * abs(scale) * terms[:, :, see].max(-1, keepdims=True)
                s = np.where(see, s, -np.inf)
                x = np.exp(s - s.max(-1, keepdims=True))
                p = x / x.sum(-1, keepdims=True)
                reach = np.abs(s[:, :, see]).max(-1, keepdims=True)
                rel = np.expm1(2 * e) + 4 * eps * reach + (16 + int(see.sum()) + nq * gqa) * eps
                total += p.sum(1)
                err += (p * rel).sum(1)
        out.append(total)
        bound.append(err + 1e-37)
    return out, bound


def scale_of(fmt):
    return 1.0 / math.sqrt(fmt.head_dim)
