"""GPU: numbers that do not fit the 32 bits of the C entry points: refused, or cut where
what they ask for is the same."""

from __future__ import annotations

import pytest

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")


@pytest.fixture(scope="module", autouse=True)
def _gpu():
    if not torch.cuda.is_available():
        pytest.skip("no GPU")


@pytest.mark.parametrize("many", [1 << 31, 1 << 32, (1 << 40) + 3])
def test_protected_tokens(many):
    from pkv import ops

    mass = torch.rand((1, 1, 100), device="cuda")
    kept, _ = ops.evict_select(mass, [100], 10, recent=many)
    assert kept[0, 0].tolist() == list(range(90, 100))
    kept, _ = ops.evict_select(mass, [100], 10, sinks=many, recent=2)
    assert kept[0, 0].tolist() == list(range(8)) + [98, 99]
    for bad in (dict(sinks=-many), dict(recent=-many)):
        with pytest.raises(ValueError):
            ops.evict_select(mass, [100], 10, **bad)


def test_beams():
    from pkv import ops

    logits, scores = torch.rand((1, 2, 50), device="cuda"), torch.zeros((1, 2), device="cuda")
    done = torch.zeros((1, 2), dtype=torch.bool, device="cuda")
    with pytest.raises(ValueError):
        ops.beam_select(logits, scores, 4, done=done, pad_token=(1 << 32) + 1)
    with pytest.raises(ValueError):
        ops.beam_select(logits, scores, (1 << 32) + 4)


def test_rows():
    """A byte tensor of more rows than 32 bits number."""
    from pkv import ops

    state = torch.zeros((1 << 32) + 16, dtype=torch.uint8, device="cuda")
    state[3] = 7
    with pytest.raises(ValueError):
        ops.reorder_rows(state, [1], [3])
    ops.reorder_rows(state[:1 << 20], [1], [3])
    assert state[:4].tolist() == [0, 7, 0, 7]
