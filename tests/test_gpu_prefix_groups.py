"""GPU: a runner takes an arena's prefix groups for the slots that they are of, as long as
these hold what they share."""

from __future__ import annotations

import pytest

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")


@pytest.fixture(scope="module", autouse=True)
def _gpu():
    if not torch.cuda.is_available():
        pytest.skip("no GPU")


def _runner():
    from pkv import ops
    from pkv.device_arena import DevicePageArena, DeviceRunner
    from pkv.layer import AttentionStack, ModelSpec

    model = AttentionStack(ModelSpec(hidden=256, query_heads=8, kv_heads=2, head_dim=64, num_layers=2,
                                     rope_theta=10000.0, dtype="bfloat16", vocab_size=100), seed=3)
    arena = DevicePageArena(ops.PageFormat(2, 64, 16, 8, 32, torch.bfloat16), 200, num_layers=2, max_slots=16,
                            max_tokens=1024)
    return DeviceRunner(model, arena)


def _hidden(rows, seed, lead=()):
    gen = torch.Generator().manual_seed(seed)
    return torch.randn((*lead, rows, 256), generator=gen).cuda().bfloat16()


def _batch(runner):
    """Two prompts of 70 and 50 tokens, two answers to each: six slots."""
    arena = runner.arena
    slots = [arena.open_slot() for _ in range(6)]
    runner.prefill(slots[:2], _hidden(120, 1), [70, 50])
    for source, slot in zip((0, 0, 1, 1), slots[2:]):
        arena.fork([slots[source]], [slot])
    return slots


def _refused(runner, slots, groups):
    x = _hidden(1, 5, (len(slots),))
    held = list(runner.arena.lengths)
    with pytest.raises(ValueError):
        runner.execute(slots, x, shared=groups)
    with pytest.raises(ValueError):
        runner.capture_decode(slots, x, shared=groups)
    assert runner.arena.lengths == held


def test_other_slots_of_the_same_count():
    runner = _runner()
    arena, slots = runner.arena, _batch(runner)
    groups = arena.prefix_groups(slots)
    assert [t.tolist() for t in groups] == [[0, 2, 3, 1, 4, 5], [0, 3, 6], [64, 48]] and len(groups) == 3
    others = [arena.open_slot() for _ in range(6)]
    arena.reserve(others, [80] * 6)
    _refused(runner, [slots[i] for i in (1, 0, 2, 3, 4, 5)], groups)
    _refused(runner, slots[::-1], groups)
    _refused(runner, others, groups)
    _refused(runner, slots[:5] + others[:1], groups)
    _refused(runner, slots[:5], groups)
    with pytest.raises(ValueError):
        arena.prefix_groups([slots[0], -1])
    with pytest.raises(ValueError):
        arena.prefix_groups([16])
    runner.execute(slots, _hidden(1, 5, (6,)), shared=groups)
    runner.execute(slots, _hidden(1, 5, (6,)), shared=tuple(groups))


def test_members_that_are_cut():
    """Truncated below what they share, released and reopened, reordered from outside, evicted."""
    runner = _runner()
    arena, slots = runner.arena, _batch(runner)
    x = _hidden(1, 5, (6,))
    groups = arena.prefix_groups(slots)
    arena.truncate([slots[0]], [64])
    runner.execute(slots, x, shared=groups)              # (holds all that is shared)
    arena.truncate([slots[2]], [63])
    _refused(runner, slots, groups)
    groups = arena.prefix_groups(slots)
    assert groups[2].tolist() == [48, 48]
    runner.execute(slots, x, shared=groups)
    # reopened with another text
    arena.release([slots[5]])
    assert arena.open_slot() == slots[5]
    arena.reserve([slots[5]], [60])
    _refused(runner, slots, groups)
    groups = arena.prefix_groups(slots)
    runner.execute(slots, x, shared=groups)
    # parents within a group, then from another one
    arena.reorder([slots[2], slots[3]], [slots[3], slots[0]])
    runner.execute(slots, x, shared=groups)
    arena.reorder([slots[2]], [slots[1]])
    _refused(runner, slots, groups)
    # evicted: below the budget nothing moves
    arena.track_mass()
    groups = arena.prefix_groups(slots)
    runner.execute(slots, x, shared=groups)
    arena.evict(slots, 500)
    runner.execute(slots, x, shared=groups)
    arena.evict(slots, 55, recent=16)
    _refused(runner, slots, groups)
    groups = arena.prefix_groups(slots)
    arena.evict(slots[:2], torch.tensor([40, 500], dtype=torch.int32, device="cuda"), max_keep=500, recent=16)
    runner.execute(slots, x, shared=groups)              # (nothing was shared any more)
    assert groups[2].tolist() == [0] * groups[2].numel()
    arena.check()


def test_a_group_that_shares_nothing_may_be_cut():
    runner = _runner()
    arena = runner.arena
    slots = [arena.open_slot() for _ in range(3)]
    runner.prefill(slots[:2], _hidden(60, 1), [30, 30])
    arena.fork([slots[0]], [slots[2]])
    groups = arena.prefix_groups(slots)
    assert sorted(groups[2].tolist()) == [0, 16]
    arena.truncate([slots[1]], [3])
    runner.execute(slots, _hidden(1, 5, (3,)), shared=groups)
    arena.truncate([slots[0]], [3])
    _refused(runner, slots, groups)


def test_a_step_that_raises_leaves_them():
    from pkv.modes import ModelCapabilityUnsupported

    runner = _runner()
    slots = _batch(runner)
    groups = runner.arena.prefix_groups(slots)
    with pytest.raises(ModelCapabilityUnsupported):      # (more query rows than a shared step takes)
        runner.execute(slots, _hidden(9, 5, (6,)), shared=groups)
    runner.execute(slots, _hidden(2, 5, (6,)), shared=groups)


def test_captured_steps():
    runner = _runner()
    arena, slots = runner.arena, _batch(runner)
    step = runner.capture_decode(slots, _hidden(1, 5, (6,)), shared=arena.prefix_groups(slots))
    step.replay()
    arena.sync_lengths()
    arena.truncate(slots, [70, 50, 70, 70, 50, 50])
    step.replay()
    arena.sync_lengths()
    arena.truncate([slots[4]], [40])
    torch.cuda.synchronize()
    held = arena.lens.tolist()
    with pytest.raises(ValueError):
        step.replay()
    assert arena.lens.tolist() == held
    arena.check()
