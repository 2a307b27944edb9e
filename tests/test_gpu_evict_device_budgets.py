"""GPU: eviction of slots named on the host by budgets on the device: the host's lengths
follow, and a slot without room is reported."""

from __future__ import annotations

import pytest

from test_gpu_cache_life import _arena, _step

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")


@pytest.fixture(scope="module", autouse=True)
def _gpu():
    if not torch.cuda.is_available():
        pytest.skip("no GPU")


def test_lengths_follow():
    arena = _arena(capacity=60, slots=5)
    a, b = arena.open_slot(), arena.open_slot()
    _step(arena, [a, b], 90, 2, torch.Generator().manual_seed(2))
    arena.evict([a, b], torch.tensor([40, 200], device="cuda"), max_keep=64)
    assert arena.lengths[a] == 40 and arena.lengths[b] == 64
    assert [arena.lengths[s] for s in range(5)] == arena.lens.tolist()
    arena.truncate([a], [40])
    arena.reserve([a, b], [100, 100])


def test_no_room_raises():
    from pkv.cache_errors import CacheCapacityError

    arena = _arena(capacity=22, slots=6)
    a, b = arena.open_slot(), arena.open_slot()
    _step(arena, [a, b], 160, 2, torch.Generator().manual_seed(1))        # 10 pages each, 2 left
    with pytest.raises(CacheCapacityError):
        arena.evict([a, b], torch.tensor([60, 60]), max_keep=60)
    assert arena.lengths[a] == arena.lengths[b] == 160 and arena.status() == (2, 0)
