"""GPU: beam selection over logits of large finite size: masks that constrained decoding
uses, whole strips and rows of them, and rows whose maximum is large."""

from __future__ import annotations

import pytest

from test_gpu_beam_select import _check, _inputs

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")


@pytest.fixture(scope="module", autouse=True)
def _gpu():
    if not torch.cuda.is_available():
        pytest.skip("no GPU")


# 8e6 is where a logit times log2(e) no longer fits an integer of float32 exactly
@pytest.mark.parametrize("low", [-7.9e6, -8.1e6, -1e9, -3e9, -1e10, -1e12, -1e20, -1e30, -1e32, -1e38, -2.3e38, -2.5e38])
@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("vocab", [700, 9001, 40001])
def test_finite_masks(dtype, vocab, low):
    """Ten tokens of a row allowed, so that most strips of the vocabulary hold masked
    ones only; a row without any; all rows of a group without any."""
    logits, scores = _inputs(3, 4, vocab, getattr(torch, dtype), 11)
    gen = torch.Generator().manual_seed(vocab)
    allowed = torch.zeros(logits.shape, dtype=torch.bool, device="cuda")
    for g in range(2):
        for w in range(4):
            allowed[g, w, torch.randperm(vocab, generator=gen)[:10].cuda()] = True
    allowed[1, 2] = False
    logits[~allowed] = low
    _check(logits, scores, 8)
    _check(logits, scores, 24)
    done = torch.zeros((3, 4), dtype=torch.bool, device="cuda")
    done[0, 1] = done[2, 0] = True
    _check(logits, scores, 8, done, 3)
    # fewer tokens allowed than are asked for: masked ones follow, the lowest first
    alone = torch.full((2, 1, vocab), low, device="cuda").to(logits.dtype)
    alone[:, 0, 5], alone[:, 0, vocab - 2] = 1.0, 2.0
    _check(alone, scores[:2, :1], 20)


@pytest.mark.parametrize("most", [7.9e6, 8.1e6, 1e9, 1e10, -1e10, 1e30, -1e30, 2e38, 3e38, -3e38])
@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
def test_large_maxima(dtype, most):
    """Rows whose largest logits are large, a few float32 steps apart."""
    gen = torch.Generator().manual_seed(3)
    step = abs(most) * 2.0 ** -23
    x = most - step * torch.randint(0, 4, (2, 3, 9001), generator=gen).double()
    low = torch.rand(x.shape, generator=gen) < 0.9
    x[low] = most - abs(most) / 2 if abs(most) < 1.5e38 else -3.3e38
    scores = -10 * torch.rand((2, 3), generator=gen).cuda()
    _check(x.float().cuda().to(getattr(torch, dtype)), scores, 16)


@pytest.mark.parametrize("most", [-6.0e4, 6.0e4])
def test_float16_masks(most):
    logits, scores = _inputs(2, 4, 9001, torch.float16, 4)
    logits[:, :, 40:] = most
    _check(logits, scores, 16)
