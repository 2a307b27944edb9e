"""GPU: operators on cached state over no queries and over no tokens."""

from __future__ import annotations

import pytest

from cache_ops_case import filled

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")


@pytest.fixture(scope="module", autouse=True)
def _gpu():
    if not torch.cuda.is_available():
        pytest.skip("no GPU")


@pytest.mark.parametrize("pages", [4, 1 << 16])
def test_attention_mass_of_no_queries(pages):
    """The sums so far go to the output as they are, under small tables and under such as
    scores are not kept for."""
    from pkv import ops

    fmt = ops.PageFormat(4, 64, 128, 8, 32, torch.bfloat16)
    lens = [300, 17, 0, 1, 256, 129, 255, 40]
    pool, table, _ = filled(fmt, lens)
    wide = torch.full((8, pages), -1, dtype=torch.int32, device="cuda")
    wide[:, :3] = table[:, :3]
    q = torch.zeros((8, 8, 0, 64), dtype=torch.bfloat16, device="cuda")
    old = torch.rand((8, 4, 512), device="cuda")
    out = torch.full((8, 4, 512), -7.0, device="cuda")
    ops.attention_mass(fmt, pool, q, wide, lens, scale=0.125, mass=old, out=out)
    for b, n in enumerate(lens):
        assert torch.equal(out[b, :, :n], old[b, :, :n])
        assert (out[b, :, n:] == -7.0).all()
