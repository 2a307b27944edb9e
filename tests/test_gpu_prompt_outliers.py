"""GPU: prompt attention beside channels of V that are far larger than the others."""

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


@pytest.mark.parametrize("dtype", ["bfloat16", "float16"])
@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("lens", [[2, 3, 5, 8, 13, 21], [1, 40, 700], [1300]])
@pytest.mark.parametrize("gain", [1.0, 4.0])
def test_large_channels(dtype, dim, lens, gain):
    """Channels of 30 for every row, of about 30, and of 1000 in one row: a weight is off by its
    rounding as an operand (2^-8 of itself at most in bfloat16, 2^-11 in float16), a channel that
    is the same everywhere by none of it, since the weights add up to one as they are rounded."""
    from pkv import ops

    dtype, rows = getattr(torch, dtype), sum(lens)
    gen = torch.Generator().manual_seed(dim + rows)
    q, k, v = (torch.randn((rows, h, dim), generator=gen) for h in (4, 2, 2))
    v[..., 3] = 30.0
    v[..., 4] = -30.0
    v[..., 5] = 30.0 + 2.0 * v[..., 5]
    v[..., 6] *= 30.0
    v[rows // 2, :, 7] = 1000.0
    q, k, v = (t.to(dtype).cuda() for t in (q * gain, k, v))
    starts = np.concatenate([[0], np.cumsum(lens)]).astype(np.int32)
    scale = dim ** -0.5
    out = ops.prompt_attention(q, k, v, torch.from_numpy(starts).cuda(), scale=scale)
    assert bool((out[..., 3] == 30.0).all()) and bool((out[..., 4] == -30.0).all())
    got, q64, k64, v64 = (t.double().cpu().numpy() for t in (out, q, k, v))
    for a, b in zip(starts, starts[1:]):
        for h in range(4):
            want, weight, terms = attention64(q64[a:b, h], k64[a:b, h // 2], v64[a:b, h // 2], np.arange(1, b - a + 1), scale)
            bound = attention_bound(want, weight, terms, scale, dtype, dim=dim, tokens=b - a, operand=half_step(dtype))
            off = np.abs(got[a:b, h] - want)
            assert np.all(off <= bound), (a, h, float((off / bound).max()))
