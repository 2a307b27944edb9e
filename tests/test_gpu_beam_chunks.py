"""GPU: beam selection on both sides of the sizes where its chunks grow, for each type,
in a workspace of just the size that is asked for."""

from __future__ import annotations

import pytest

from test_gpu_beam_select import _check, _inputs

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")


@pytest.fixture(scope="module", autouse=True)
def _gpu():
    if not torch.cuda.is_available():
        pytest.skip("no GPU")


# 2 chunks of 8192 a row: 1008 and 1024 of them, 496 and 512 candidates of a group, 8064 and 8192
@pytest.mark.parametrize("groups,beams,count", [(126, 4, 64), (128, 4, 64), (128, 4, 62), (8, 64, 63), (8, 64, 64)])
@pytest.mark.parametrize("dtype", ["float32", "bfloat16", "float16"])
def test_sizes(dtype, groups, beams, count):
    from pkv import _native, ops

    logits, scores = _inputs(groups, beams, 9001, getattr(torch, dtype), count)
    logits[1] = 0
    logits[2, :, :8990] = -1e4
    logits[3, 1, 5] = float("nan")
    _check(logits, scores, count)
    want = ops.beam_select(logits, scores, count)
    size = _native.load().pkv_beam_workspace_bytes(groups, beams, 9001, count)
    guarded = torch.full((size + 4096,), 77, dtype=torch.uint8, device="cuda")
    got = ops.beam_select(logits, scores, count, workspace=guarded[:size])
    assert all(torch.equal(x, y) for x, y in zip(want, got))
    assert (guarded[size:] == 77).all()
