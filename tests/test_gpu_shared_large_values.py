"""GPU: attention over shared prefixes where quantized pages hold values past float16's range
(a group's scale and bias are float16 numbers; bias + 255 scale may be beyond)."""

from __future__ import annotations

import numpy as np
import pytest

from step_case import paged64, side64
from test_gpu_shared_attention import _cache, _format, _queries

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")


@pytest.fixture(scope="module", autouse=True)
def _gpu():
    if not torch.cuda.is_available():
        pytest.skip("no GPU")


def _put(fmt, pool, table, at, value):
    """Store tokens ``at = [(sequence, position), ...]`` with V ``value(i) [HK, D]``."""
    from pkv import ops

    for i, (b, t) in enumerate(at):
        batch = table.shape[0]
        side = torch.zeros((2, batch, fmt.num_kv_heads, 1, fmt.head_dim))
        side[0] = torch.randn(side[0].shape, generator=torch.Generator().manual_seed(i))
        side[1] = value(i)[:, None]
        side = side.to(fmt.dtype).cuda()
        ops.append_quantize(fmt, pool, side[0].contiguous(), side[1].contiguous(), table,
                            torch.full((batch,), t, dtype=torch.int32), [int(x == b) for x in range(batch)])


def _compare(fmt, pool, table, lens, members, starts, prefix, q, scale=0.1):
    from pkv import ops

    want, bound = paged64(fmt, pool, table, lens, q, scale)
    got = ops.shared_prefix_attention(fmt, pool, q, table, lens, members, starts, prefix, scale=scale)
    off = np.abs(got.double().cpu().numpy() - want)
    assert np.all(off <= bound), (float(np.nanmax(off / bound)), np.argwhere(~(off <= bound))[0].tolist())
    return want


@pytest.mark.parametrize("bits,dim,group", [(8, 64, 32), (8, 128, 64), (8, 128, 128), (8, 256, 64), (8, 80, 32),
                                            (4, 64, 64), (4, 128, 32), (4, 256, 128)])
@pytest.mark.parametrize("gqa,nq", [(4, 1), (8, 1), (4, 4)])
def test_values_past_float16(bits, dim, group, gqa, nq):
    """A maximum of 76,500, of about a million, of the most that a finite scale takes, a minimum
    below zero; in shared tokens, in a sequence's own, in the last tile and far from it;
    beside groups of ordinary values."""
    fmt = _format(bits, dim, group)
    pool, table, lens, members, starts, prefix = _cache(fmt, [(640, [300, 20, 5]), (64, [1, 40])])
    first, second = members[0], members[1]
    gen = torch.Generator().manual_seed(dim)
    most = 65000.0 * (2 ** bits - 1)

    def value(i):
        x = torch.randn((2, dim), generator=gen)
        top = (76500.0, 9e5, most, 1e5, 76500.0)[i]
        low = (0.0, 0.0, 0.0, -6e4, 0.0)[i]
        x[:, :16] = low + (top - low) * torch.rand((2, 16), generator=gen)
        x[:, 3], x[:, 7] = top, low
        return x

    _put(fmt, pool, table, [(first, 5), (first, 333), (first, 700), (second, 641), (first, 939)], value)
    held = side64(fmt, pool, table[first, :59].tolist(), True)[:, :940]    # (as many tokens as it has)
    assert np.isfinite(held).all() and held.max() > 0.9 * most
    want = _compare(fmt, pool, table, lens, members, starts, prefix, _queries(fmt, table.shape[0], gqa, nq))
    assert np.abs(want).max() > 1000


def test_many_members():
    """The same where the call is laid out by a plan."""
    fmt = _format(8, 64, 32, 16, 1)
    pool, table, lens, members, starts, prefix = _cache(fmt, [(200, [1 + 7 * i % 40 for i in range(70)])])
    _put(fmt, pool, table, [(members[0], 50), (members[40], 201)], lambda i: torch.linspace(0, 2e5, 32).repeat(2)[None])
    _compare(fmt, pool, table, lens, members, starts, prefix, _queries(fmt, 70, 4, 1))


@pytest.mark.parametrize("bits", [4, 8])
@pytest.mark.parametrize("gqa", [2, 8])
def test_rows_that_do_not_see_it(bits, gqa):
    """A later token's large values change nothing for a row before it, nor for another
    sequence."""
    from pkv import ops

    fmt = _format(bits, 128, 64)
    pool, table, lens, members, starts, prefix = _cache(fmt, [(64, [300, 40, 8])])
    nq = 4
    q = _queries(fmt, 3, gqa, nq)
    call = lambda: ops.shared_prefix_attention(fmt, pool, q, table, lens, members, starts, prefix, scale=0.1)
    clean = call()
    b = members[0]
    _put(fmt, pool, table, [(b, int(lens[b]) - 2)], lambda i: torch.linspace(-100, 1e5, 128)[None].expand(2, 128))
    got = call()
    others = [i for i in range(3) if i != b]
    assert torch.equal(got[others], clean[others])
    assert torch.equal(got[b, :, :nq - 2], clean[b, :, :nq - 2])
    assert not torch.equal(got[b, :, nq - 2:], clean[b, :, nq - 2:])
    _compare(fmt, pool, table, lens, members, starts, prefix, q)


def test_beside_infinities():
    """An infinity that a row sees stays one beside large finite values."""
    fmt = _format(8, 128, 64)
    pool, table, lens, members, starts, prefix = _cache(fmt, [(640, [300, 20])])
    first = members[0]
    x = torch.linspace(0, 1e5, 128)[None].expand(2, 128).clone()
    _put(fmt, pool, table, [(first, 5)], lambda i: x)
    x[:, 100] = float("inf")
    _put(fmt, pool, table, [(first, 800)], lambda i: x)
    from pkv import ops

    q = _queries(fmt, 2, 4, 1)
    got = ops.shared_prefix_attention(fmt, pool, q, table, lens, members, starts, prefix, scale=0.1)
    want, bound = paged64(fmt, pool, table, lens, q, 0.1)
    fine = np.isfinite(want)
    assert fine[members[1]].all() and not fine[first].all() and fine[first, :, :, :64].all()
    off = np.abs(got.double().cpu().numpy() - want)
    assert np.all(off[fine] <= bound[fine])
    assert not bool(torch.isfinite(got).cpu().numpy()[~fine].any())
