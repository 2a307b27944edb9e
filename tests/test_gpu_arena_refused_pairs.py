"""GPU: forks and truncations that the arena refuses on the device leave the slots'
attention sums and counts of evicted tokens as they were."""

from __future__ import annotations

import pytest

from test_gpu_cache_life import _arena, _step

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")


@pytest.fixture(scope="module", autouse=True)
def _gpu():
    if not torch.cuda.is_available():
        pytest.skip("no GPU")


def _i32(*x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


def _evicted_arena():
    arena = _arena(slots=6)
    slots = [arena.open_slot() for _ in range(3)]
    _step(arena, slots, 90, 2, torch.Generator().manual_seed(2))
    arena.evict(slots, [40, 60, 90])
    return arena


def test_refused_forks():
    """A destination that holds tokens, a slot that does not exist, a slot onto itself,
    between pairs that are accepted."""
    from pkv.cache_errors import CacheCorruptionError

    arena = _evicted_arena()
    mass, evicted = arena.mass.clone(), arena.evicted.clone()
    table = arena.table.clone()
    arena.fork(_i32(0, 0, 9, 1, 3, 2), _i32(4, 1, 2, 5, 3, -1))
    for source, to in ((0, 4), (1, 5)):
        assert torch.equal(arena.mass[:, to], mass[:, source])
        assert arena.evicted[to] == evicted[source] and arena.lens[to] == arena.lens[source]
    for s in (0, 1, 2, 3):
        assert torch.equal(arena.mass[:, s], mass[:, s]) and arena.evicted[s] == evicted[s]
    assert torch.equal(arena.table[:4], table[:4])
    with pytest.raises(CacheCorruptionError):
        arena.check()


def test_refused_truncations():
    from pkv.cache_errors import CacheCorruptionError

    arena = _evicted_arena()
    arena.truncate(_i32(0, 1, 2, 7), _i32(-1, 61, 0, 0))
    assert arena.evicted[:3].tolist() == [50, 30, 0] and arena.lens[:3].tolist() == [40, 60, 0]
    with pytest.raises(CacheCorruptionError):
        arena.check()
