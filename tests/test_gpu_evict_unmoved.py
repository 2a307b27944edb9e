"""GPU: evictions that are refused, fail on the way or have nothing to cut: no page is
lost, and no slot is handed out that holds tokens."""

from __future__ import annotations

import pytest

from test_gpu_cache_life import Model, _arena, _step

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")


@pytest.fixture(scope="module", autouse=True)
def _gpu():
    if not torch.cuda.is_available():
        pytest.skip("no GPU")


def _held():
    arena = _arena(capacity=60, slots=5)
    a, b = arena.open_slot(), arena.open_slot()
    _step(arena, [a, b], 90, 2, torch.Generator().manual_seed(2))
    model = Model(arena)
    model.take([a, b])
    return arena, a, b, model


def _unchanged(arena, a, b, model, free, mass):
    assert arena.status() == (free, 0)
    assert torch.equal(arena.mass, mass) and not arena.evicted.any()
    model.check([a, b])
    empty = [arena.open_slot() for _ in range(3)]
    assert arena.lens[empty].tolist() == [0, 0, 0]
    arena.reserve(empty, [0, 0, 0])
    arena.release(empty)


@pytest.mark.parametrize("bad", [dict(sinks=-1), dict(recent=-1)])
def test_refused(bad):
    arena, a, b, model = _held()
    free, mass = arena.status()[0], arena.mass.clone()
    with pytest.raises(ValueError):
        arena.evict([a, b], 40, **bad)
    _unchanged(arena, a, b, model, free, mass)


@pytest.mark.parametrize("keep", [10 ** 6, [10 ** 6, 90], [256, 257], 10 ** 12])
def test_budgets_past_the_arenas_tokens_cut_nothing(keep):
    arena, a, b, model = _held()
    free, mass = arena.status()[0], arena.mass.clone()
    arena.evict([a, b], keep)
    _unchanged(arena, a, b, model, free, mass)


def test_one_budget_past_the_arenas_tokens():
    arena, a, b, model = _held()
    model.evict([a], 40, 4, 16)
    arena.evict([a, b], [40, 10 ** 6], sinks=4, recent=16)
    model.check([a, b])
    assert arena.lengths[a] == 40 and arena.lengths[b] == 90
    assert arena.evicted[[a, b]].tolist() == [50, 0]


@pytest.mark.parametrize("call", ["evict_select", "evict_pages"])
@pytest.mark.parametrize("own_spare", [False, True])
def test_a_failure_on_the_way_gives_the_pages_back(call, own_spare, monkeypatch):
    from pkv import ops

    arena, a, b, model = _held()
    free = arena.status()[0]
    spare = [arena.open_slot()] if own_spare else None

    def fails(*_a, **_k):
        raise MemoryError(call)

    with monkeypatch.context() as patch:
        patch.setattr(ops, call, fails)
        with pytest.raises(MemoryError):
            arena.evict([a, b], 40, spare=spare)
    assert arena.status() == (free, 0) and not arena.evicted.any()
    model.check([a, b])
    assert not arena.lens[2:].any()
    arena.evict([a, b], 40, spare=spare)
    assert arena.lens[:2].tolist() == [40, 40]


def test_a_failure_after_some_slots_were_cut(monkeypatch):
    """With one spare slot the slots are cut one after the other: the host's lengths are
    those of the device whichever of them fails."""
    from pkv import ops

    arena, a, b, model = _held()
    spare = [arena.open_slot()]
    works, calls = ops.evict_select, []

    def fails_second(*args, **kw):
        calls.append(1)
        if len(calls) == 2:
            raise MemoryError("the second slot")
        return works(*args, **kw)

    model.evict([a], 40, 4, 64)
    with monkeypatch.context() as patch:
        patch.setattr(ops, "evict_select", fails_second)
        with pytest.raises(MemoryError):
            arena.evict([a, b], 40, spare=spare)
    assert arena.lengths[a] == 40 and arena.lengths[b] == 90
    assert arena.lengths == arena.lens.tolist() and arena.evicted[[a, b]].tolist() == [50, 0]
    model.check([a, b])


@pytest.mark.parametrize("call", ["_scratch", "evict_select"])
def test_no_memory_for_a_call_leaves_the_sums(call, monkeypatch):
    """Memory is taken before the sums move: without any, nothing has."""
    from pkv import ops

    arena, a, b, model = _held()
    free, mass = arena.status()[0], arena.mass.clone()

    def fails(*_a, **_k):
        raise MemoryError(call)

    with monkeypatch.context() as patch:
        patch.setattr(ops, call, fails)
        with pytest.raises(MemoryError):
            arena.evict([a, b], 40)
    _unchanged(arena, a, b, model, free, mass)
