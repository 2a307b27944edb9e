"""GPU: errors that the device arena holds from earlier calls outlive an eager step that raises."""

from __future__ import annotations

from types import SimpleNamespace

import pytest

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")


@pytest.fixture(scope="module", autouse=True)
def _gpu():
    if not torch.cuda.is_available():
        pytest.skip("no GPU")


class _Raises:
    """A model whose forward raises."""

    spec = SimpleNamespace(num_layers=1)

    def forward(self, hidden, *, cache, position_ids):
        raise RuntimeError("the model's own")


def _arena():
    from pkv import ops
    from pkv.device_arena import DevicePageArena

    return DevicePageArena(ops.PageFormat(2, 64, 16, 8, 32, torch.bfloat16), 6, max_slots=8, max_tokens=512)


def _unread_error(arena, slot):
    """What a captured step records without pages: nobody has read it yet."""
    arena.reserve(torch.tensor([slot], dtype=torch.int32, device="cuda"),
                  torch.tensor([400], dtype=torch.int32, device="cuda"))


@pytest.mark.parametrize("prefill", [False, True])
def test_an_earlier_error_stays(prefill):
    from pkv.cache_errors import CacheCapacityError, CacheCorruptionError
    from pkv.device_arena import CORRUPT, OUT_OF_PAGES, DeviceRunner

    arena = _arena()
    runner = DeviceRunner(_Raises(), arena)
    a, b = arena.open_slot(), arena.open_slot()

    def step(tokens):
        with pytest.raises(RuntimeError, match="the model's own"):
            if prefill:
                runner.prefill([a], torch.zeros((tokens, 8), device="cuda"), [tokens])
            else:
                runner.execute([a], torch.zeros((1, tokens, 8), device="cuda"))
        assert arena.lengths[a] == 0 and int(arena.lens[a]) == 0

    # nothing recorded before: a failed reserve's record goes with its step
    for tokens in (5, 200):
        step(tokens)
        assert arena.check() == 6
    # recorded before: it is still there, after a step that has its pages and one that has not
    for tokens in (5, 200):
        _unread_error(arena, b)
        step(tokens)
        with pytest.raises(CacheCapacityError):
            arena.check()
        assert arena.check() == 6
        arena.state[1:2].fill_(CORRUPT)
        step(tokens)
        assert arena.status()[1] == CORRUPT
        with pytest.raises(CacheCorruptionError):
            arena.check()
        arena.state[1:2].fill_(CORRUPT | OUT_OF_PAGES)
        step(tokens)
        assert arena.status()[1] == CORRUPT | OUT_OF_PAGES
        arena.state[1:2].zero_()


class _Gives:
    """A model that gives its input back."""

    spec = SimpleNamespace(num_layers=1)

    def forward(self, hidden, *, cache, position_ids):
        return hidden


def test_a_step_that_raises_an_earlier_error():
    """The step's own slots are as they were, on the device as well: those whose reserve
    succeeded, and those of a reserve without pages."""
    from pkv.cache_errors import CacheCapacityError
    from pkv.device_arena import DeviceRunner

    arena = _arena()
    runner = DeviceRunner(_Gives(), arena)
    a, b = arena.open_slot(), arena.open_slot()
    runner.execute([a], torch.zeros((1, 20, 8), device="cuda"))
    for tokens in (5, 40, 200):
        for earlier in (True, False):
            if earlier:
                _unread_error(arena, b)
            elif tokens < 200:
                continue
            with pytest.raises(CacheCapacityError):
                runner.execute([a], torch.zeros((1, tokens, 8), device="cuda"))
            assert arena.check() == 4 and arena.lengths[a] == int(arena.lens[a]) == 20
    runner.execute([a], torch.zeros((1, 5, 8), device="cuda"))
    assert arena.check() == 4 and arena.lengths[a] == int(arena.lens[a]) == 25


@pytest.mark.parametrize("model", [_Raises, _Gives])
def test_a_step_that_raises_after_replays(model):
    """Tokens that a captured step appended, which the host's lengths do not know of, stay."""
    from pkv.device_arena import DeviceRunner

    arena = _arena()
    runner = DeviceRunner(model(), arena)
    a, b = arena.open_slot(), arena.open_slot()
    arena.reserve([a], [10])
    # (as a replay reserves: by device tensors)
    one = torch.ones(1, dtype=torch.int32, device="cuda")
    for _ in range(3):
        arena.reserve(torch.tensor([a], dtype=torch.int32, device="cuda"), one)
    if model is _Gives:
        _unread_error(arena, b)
    with pytest.raises(Exception):
        runner.execute([a], torch.zeros((1, 4, 8), device="cuda"))
    assert int(arena.lens[a]) == 13 and arena.lengths[a] == 10
    arena.sync_lengths()
    assert arena.lengths[a] == 13 and arena.check() == 5
