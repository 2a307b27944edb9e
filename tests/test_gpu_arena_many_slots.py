"""GPU: evictions and forks of more slots than one kernel call takes."""

from __future__ import annotations

import numpy as np
import pytest

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")


@pytest.fixture(scope="module", autouse=True)
def _gpu():
    if not torch.cuda.is_available():
        pytest.skip("no GPU")


def _arena(slots, capacity):
    from pkv import ops
    from pkv.device_arena import DevicePageArena

    arena = DevicePageArena(ops.PageFormat(1, 64, 16, 8, 32, torch.bfloat16), capacity, max_slots=slots, max_tokens=64)
    arena.track_mass()
    gen = torch.Generator(device="cuda").manual_seed(1)
    arena.mass.copy_(torch.rand(arena.mass.shape, generator=gen, device="cuda"))
    arena.pools[0].copy_(torch.randint(0, 256, arena.pools[0].shape, generator=gen, device="cuda", dtype=torch.uint8))
    return arena


def test_eviction():
    """4100 slots at once: each slot's kept sums, lengths and pages."""
    from test_gpu_evict import _plain, _tokens

    arena = _arena(8300, 13000)
    slots = [arena.open_slot() for _ in range(4100)]
    arena.reserve(slots, [20] * len(slots))
    before = {s: [x[:, :20] for x in _tokens(arena.fmt, arena.pools[0], arena.pages(s))] for s in slots[::500] + slots[-3:]}
    mass = arena.mass[0, :, 0].cpu().numpy()
    arena.evict(slots, 10, sinks=1, recent=3)
    assert arena.status()[1] == 0 and set(arena.lens[slots].tolist()) == {10}
    after = arena.mass[0, :, 0].cpu().numpy()
    for s in slots:
        assert np.array_equal(after[s, :10], mass[s][_plain(mass[s], 20, 10, 1, 3)])
    for s, held in before.items():
        kept = _plain(mass[s], 20, 10, 1, 3)
        for x, y in zip(_tokens(arena.fmt, arena.pools[0], arena.pages(s)), held):
            assert np.array_equal(x[:, :10], y[:, kept])
    arena.release(slots)
    assert arena.status() == (13000, 0)


def test_fork():
    arena = _arena(16500, 13000)
    slots = [arena.open_slot() for _ in range(16400)]
    heads, others = slots[:8200], slots[8200:]
    arena.reserve(heads, [5] * len(heads))
    mass = arena.mass.clone()
    arena.fork(heads, others)
    assert arena.status()[1] == 0 and set(arena.lens[others].tolist()) == {5}
    assert torch.equal(arena.mass[:, others], mass[:, heads]) and torch.equal(arena.mass[:, heads], mass[:, heads])
