"""GPU: attention over shared prefixes where one token outweighs a long tail of equal ones,
whose weights are far below the largest."""

from __future__ import annotations

import numpy as np
import pytest

from shared_bound import shared64

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")


@pytest.fixture(scope="module", autouse=True)
def _gpu():
    if not torch.cuda.is_available():
        pytest.skip("no GPU")


@pytest.mark.parametrize("gap", [7.5, 18.4, 22.3, 25.6])
@pytest.mark.parametrize("bits,dim,group", [(8, 64, 32), (4, 128, 64), (8, 128, 128), (16, 64, 32), (16, 128, 32),
                                            (8, 256, 64), (16, 256, 32)])
@pytest.mark.parametrize("dtype", ["float16", "bfloat16"])
@pytest.mark.parametrize("top", [5, 900, 1050])
@pytest.mark.parametrize("gqa", [1, 8])
def test_a_tail_far_below_one_token(gap, bits, dim, group, dtype, top, gqa):
    """The token at ``top`` is 2^gap above the others (its value zero, theirs about 100), a
    shared one or each sequence's own.  Weights carry their operands' rounding; float16 ones
    have a fixed step of 2^-31 of the largest, half of it an error per token."""
    from pkv import ops

    dtype, batch, shared, n = getattr(torch, dtype), 4, 1024, 1100
    fmt = ops.PageFormat(1, dim, 16, bits, group, dtype)
    gen = torch.Generator().manual_seed(dim)
    k = torch.zeros((batch, 1, n, dim))
    k[:, 0, top, 0] = gap / 4.0
    v = 100.0 + torch.randn((1, 1, n, dim), generator=gen).expand(batch, 1, n, dim).clone()
    v[:, :, top] = 0.0
    pages = -(-n // 16)
    table = np.arange(batch * pages, dtype=np.int32).reshape(batch, pages)
    table[:, :shared // 16] = table[0, :shared // 16]
    table = torch.from_numpy(table).cuda()
    pool = ops.allocate_pool(fmt, batch * pages)
    lens = torch.tensor([1100, 1099, 1060, 1075], dtype=torch.int32, device="cuda")
    ops.append_quantize(fmt, pool, k.to(dtype).cuda(), v.to(dtype).cuda(), table, torch.zeros_like(lens), lens)
    q = torch.zeros((batch, gqa, 1, dim), dtype=dtype, device="cuda")
    q[..., 0] = 4.0
    scale = 0.6931471805599453    # (scores in powers of two)
    want, bound = shared64(fmt, pool, table, lens, q, scale)
    got = ops.shared_prefix_attention(fmt, pool, q, table, lens, list(range(batch)), [0, batch], [shared], scale=scale)
    off = np.abs(got.double().cpu().numpy() - want)
    assert np.all(off <= bound), float((off / bound).max())
