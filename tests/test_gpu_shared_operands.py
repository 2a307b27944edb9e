"""GPU: what attention over shared prefixes says of its operands -- quantized keys enter as
they are, weights as two operands where one would show -- on inputs where a rounding of
either would stand out, beside the same computed with that rounding."""

from __future__ import annotations

import numpy as np
import pytest

from shared_bound import shared64
from step_case import side64

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")


@pytest.fixture(scope="module", autouse=True)
def _gpu():
    if not torch.cuda.is_available():
        pytest.skip("no GPU")


def _cache(fmt, k, v, batch, shared):
    """``k, v [tokens, D]`` in every sequence, the first ``shared`` tokens on the same pages."""
    from pkv import ops

    n, dim = k.shape
    pages = -(-n // 16)
    table = np.arange(batch * pages, dtype=np.int32).reshape(batch, pages)
    table[:, :shared // 16] = table[0, :shared // 16]
    table = torch.from_numpy(table).cuda()
    pool = ops.allocate_pool(fmt, batch * pages)
    sides = [t.to(fmt.dtype).cuda().view(1, 1, n, dim).expand(batch, 1, n, dim).contiguous() for t in (k, v)]
    lens = torch.full((batch,), n, dtype=torch.int32, device="cuda")
    ops.append_quantize(fmt, pool, *sides, table, torch.zeros_like(lens), lens)
    return pool, table, lens


def _softmax(x):
    p = np.exp(x - x.max())
    return p / p.sum()


@pytest.mark.parametrize("bits", [4, 8])
@pytest.mark.parametrize("dim,group", [(64, 32), (128, 64), (128, 128), (256, 64)])
@pytest.mark.parametrize("gqa", [2, 12])
def test_keys_as_their_codes(bits, dim, group, gqa):
    """Keys between 1 and 1 + 2^-10, where float16 has nothing between: as float16 operands they
    would be off by as much, all in one direction."""
    from pkv import ops

    fmt = ops.PageFormat(1, dim, 16, bits, group, torch.float16)
    batch, shared, n = 3, 64, 90
    k = torch.ones((n, dim))
    k[:, ::group] += 2.0 ** -10                       # (the group's largest: codes are between)
    v = (-1.0) ** torch.arange(n)[:, None].expand(n, dim)
    pool, table, lens = _cache(fmt, k, v, batch, shared)
    # a page's codes are its own: every other token has codes past the middle
    pages = sorted({int(x) for x in table.flatten()})
    size = fmt.page_bytes
    for page in pages:
        held = pool[page].clone()
        payload = size // 2 - 16 * (fmt.stored_dim // group) * 4     # (K's tile; one KV head, 16 tokens a page)
        lane = torch.arange(payload, device="cuda") // min(16, fmt.stored_dim * bits // 32) % 64
        held[:payload] = torch.where(lane % 2 == 1, 0xA0 if bits == 8 else 0xAA, 0).to(torch.uint8)
        pool[page] = held
    q = torch.full((batch, gqa, 1, dim), 4.0, dtype=torch.float16, device="cuda")
    scale = 16.0 / dim ** 0.5
    want, bound = shared64(fmt, pool, table, lens, q, scale)
    got = ops.shared_prefix_attention(fmt, pool, q, table, lens, list(range(batch)), [0, batch], [shared], scale=scale)
    off = np.abs(got.double().cpu().numpy() - want)
    assert np.all(off <= bound), float((off / bound).max())
    # rounded keys would show
    ids = table[0].tolist()
    keys, values = side64(fmt, pool, ids, False)[0, :n], side64(fmt, pool, ids, True)[0, :n]
    rounded = keys.astype(np.float16).astype(np.float64)
    assert (rounded != keys).any()
    other = _softmax(4.0 * rounded.sum(-1) * scale) @ values
    assert (np.abs(other - want[0, 0, 0]) > bound[0, 0, 0]).any()


@pytest.mark.parametrize("bits,dtype", [(4, "float16"), (8, "float16"), (16, "bfloat16")])
@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("gqa", [2, 12])
@pytest.mark.parametrize("gap", [1.7, 2.9, 4.7])
def test_weights_as_two_operands(bits, dtype, dim, gqa, gap):
    """One token against the others with the opposite sign: what is left of them is small beside
    a rounding of the others' weight, the same for all of them."""
    from pkv import ops

    dtype = getattr(torch, dtype)
    fmt = ops.PageFormat(1, dim, 16, bits, 32, dtype)
    batch, shared, n = 3, 64, 81
    k = torch.zeros((n, dim))
    q = torch.zeros((batch, gqa, 1, dim), dtype=dtype, device="cuda")
    k[7], q[..., 0] = 1.0, 1.0
    scale = gap * float(np.log(2.0))
    v = torch.full((n, dim), -8.0)
    v[7] = torch.tensor((n - 1) * 8.0 * 2.0 ** -gap).half().to(dtype).float()
    pool, table, lens = _cache(fmt, k, v, batch, shared)
    values = side64(fmt, pool, table[0].tolist(), True)[0, :n]
    assert np.array_equal(values, v.double().numpy())    # (float16 holds them: no rounding)
    want, bound = shared64(fmt, pool, table, lens, q, scale, values=0.0, products=1)
    got = ops.shared_prefix_attention(fmt, pool, q, table, lens, list(range(batch)), [0, batch], [shared], scale=scale)
    off = np.abs(got.double().cpu().numpy() - want)
    assert np.all(off <= bound), float((off / bound).max())
    # one operand would show
    p = torch.full((n,), 2.0 ** -gap, dtype=torch.float64)
    p[7] = 1.0
    p = p.to(torch.float16 if fmt.quantized else torch.bfloat16).double().numpy()
    assert (np.abs(p @ values / p.sum() - want[0, 0, 0]) > bound[0, 0, 0]).all()
