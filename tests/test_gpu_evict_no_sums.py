"""GPU: eviction over rows without any token."""

from __future__ import annotations

import pytest

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")


@pytest.fixture(scope="module", autouse=True)
def _gpu():
    if not torch.cuda.is_available():
        pytest.skip("no GPU")


@pytest.mark.parametrize("rows", [None, [1, -1]])
@pytest.mark.parametrize("shape", [(2, 3, 0), (2, 2, 3, 0)])
def test_select(shape, rows):
    from pkv import ops

    mass = torch.zeros(shape, device="cuda")
    kept, n, sums = ops.evict_select(mass, [0, 0], 5, sinks=1, recent=2, rows=rows, with_mass=True)
    assert kept.shape == (*shape[:-3], 2, 3, 5) and (kept == -1).all()
    assert n.tolist() == [0, 0]
    assert sums.shape == (*shape[:-1], 5) and not sums.any()
