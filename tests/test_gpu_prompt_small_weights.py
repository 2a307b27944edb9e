"""GPU: prompt attention where one key outweighs a long tail of equal ones, whose weights are
far below the largest."""

from __future__ import annotations

import numpy as np
import pytest

from step_case import attention64, attention_bound, half_step

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")


@pytest.fixture(scope="module", autouse=True)
def _gpu():
    if not torch.cuda.is_available():
        pytest.skip("no GPU")


@pytest.mark.parametrize("gap", [7.5, 13.7, 18.4, 22.3, 25.6])
@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("dtype", ["float16", "bfloat16"])
@pytest.mark.parametrize("top", [0, 1, 40, 2000])
def test_a_tail_far_below_one_key(gap, dim, dtype, top):
    """The key at ``top`` is 2^gap above the others (its value zero, theirs 100 and more): the
    result is the tail's, a fraction of it.  Weights carry their operand's relative rounding
    down to 2^-21 of the largest, below it a step of 2^-31 of that (half of it per token)."""
    from pkv import ops

    dtype, n = getattr(torch, dtype), 4100
    gen = torch.Generator().manual_seed(dim)
    q, k = torch.zeros((n, 2, dim)), torch.zeros((n, 1, dim))
    q[..., 0] = 4.0
    k[top, 0, 0] = gap / 4.0
    k[:, 0, 1:] = torch.randn((n, dim - 1), generator=gen)    # (met by zeros)
    v = 100.0 + torch.randn((n, 1, dim), generator=gen)
    v[top] = 0.0
    q, k, v = (t.to(dtype).cuda() for t in (q, k, v))
    scale = 0.6931471805599453    # (scores in powers of two)
    got = ops.prompt_attention(q, k, v, [0, n], scale=scale).double().cpu().numpy()
    pick = np.array([top, top + 1, top + 31, top + 64, 2050, 3000, 4099])
    q64, k64, v64 = (t.double().cpu().numpy() for t in (q, k, v))
    for h in range(2):
        want, weight, terms = attention64(q64[pick, h], k64[:, 0], v64[:, 0], pick + 1, scale)
        bound = attention_bound(want, weight, terms, scale, dtype, dim=dim, tokens=n, operand=half_step(dtype))
        if dtype is torch.float16:
            bound += (pick + 1)[:, None] * 2.0 ** -32 * np.abs(v64).max()
        off = np.abs(got[pick, h] - want)
        assert np.all(off <= bound), (h, float((off / bound).max()))
