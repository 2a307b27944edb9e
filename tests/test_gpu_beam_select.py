"""GPU: a beam step's selection over beams and vocabulary, against a plain one in 64
bits on the host."""

from __future__ import annotations

import math

import pytest

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")


@pytest.fixture(scope="module", autouse=True)
def _gpu():
    if not torch.cuda.is_available():
        pytest.skip("no GPU")


def _plain(logits, scores, count, done=None, pad=0):
    x = logits.double().cpu()
    scores = scores.double().cpu()
    # the maximum apart: where it is the type's lowest value it would swallow the sum
    most = x.amax(-1, keepdim=True)
    lse = torch.exp(x - most).sum(-1, keepdim=True).log()
    c = scores[..., None] - lse + (x - most)
    c[~torch.isfinite(lse + most)[..., 0]] = -math.inf
    if done is not None:
        for g, w in done.cpu().nonzero().tolist():
            c[g, w] = -math.inf
            c[g, w, pad] = scores[g, w]
    c[~torch.isfinite(scores)] = -math.inf
    best = torch.sort(c.flatten(1), dim=1, descending=True, stable=True)
    flat = best.indices[:, :count]
    return best.values[:, :count], flat // logits.shape[2], flat % logits.shape[2]


def _check(logits, scores, count, done=None, pad=0):
    from pkv import ops

    got = ops.beam_select(logits, scores, count, done=done, pad_token=pad)
    want = _plain(logits, scores, count, done, pad)
    assert torch.equal(got[1].cpu().long(), want[1])
    assert torch.equal(got[2].cpu().long(), want[2])
    # the score is rounded to float32 once; a float32 exponential of x - max is off by
    # 2^-22 of itself, and by the rounding of its scaled argument, |x - max| 2^-23, which
    # the log-sum-exp takes over weighted by softmax; blocks of 64 float32 sums add 2^-21
    live = torch.isfinite(want[0])
    assert torch.equal(torch.isfinite(got[0].cpu()), live)
    off = (got[0].cpu().double() - want[0]).abs()
    x = logits.double().cpu()
    reach = (torch.softmax(x, -1) * (x.amax(-1, keepdim=True) - x)).nan_to_num(0, 0, 0).sum(-1).amax(1, keepdim=True)
    assert (off <= 2.0 ** -24 * want[0].abs() + 2.0 ** -23 * reach + 2.0 ** -21)[live].all()
    assert (got[0].cpu()[~live] == -math.inf).all()


def _inputs(groups, beams, vocab, dtype, seed=0):
    gen = torch.Generator().manual_seed(seed)
    x = torch.randn((groups, beams, vocab), generator=gen) * 3
    return x.cuda().to(dtype), -10 * torch.rand((groups, beams), generator=gen).cuda()


@pytest.mark.parametrize("dtype", ["float32", "bfloat16", "float16"])
@pytest.mark.parametrize("groups,beams,vocab,count", [
    (1, 1, 1, 1), (1, 1, 2, 2), (2, 3, 7, 5), (1, 1, 64, 64), (3, 4, 63, 8), (2, 5, 1000, 10), (5, 2, 1023, 4),
    (1, 4, 32000, 8), (2, 16, 4099, 32), (1, 64, 300, 64), (4, 8, 2047, 16), (2, 3, 128256, 6), (1, 1, 200000, 1),
    (7, 6, 8193, 12)])
def test_shapes(dtype, groups, beams, vocab, count):
    logits, scores = _inputs(groups, beams, vocab, getattr(torch, dtype), vocab + count)
    _check(logits, scores, count)
    done = torch.rand((groups, beams), generator=torch.Generator().manual_seed(count)).cuda() < 0.4
    _check(logits, scores, count, done, vocab - 1)


@pytest.mark.parametrize("dtype", ["float32", "bfloat16", "float16"])
@pytest.mark.parametrize("vocab", [97, 5000, 40001])
def test_ties(dtype, vocab):
    """Equal logits, in rows and across beams of equal score: the lowest pair first."""
    dtype = getattr(torch, dtype)
    scores = torch.zeros((1, 3), device="cuda")
    _check(torch.zeros((1, 3, vocab), device="cuda", dtype=dtype), scores, 64)
    gen = torch.Generator().manual_seed(1)
    few = torch.randint(0, 3, (2, 4, vocab), generator=gen).cuda().to(dtype)
    _check(few, torch.rand((2, 4), generator=gen).cuda(), 40)
    # equal rows: every pair of beams ties at every token
    row = torch.randn((1, 1, vocab), generator=gen).cuda().to(dtype)
    _check(row.expand(1, 3, vocab).contiguous(), scores, 30)
    _check(row.expand(1, 3, vocab), scores, 30)


@pytest.mark.parametrize("dtype", ["float32", "bfloat16", "float16"])
@pytest.mark.parametrize("vocab", [50, 9001])
def test_banned_tokens_and_dead_beams(dtype, vocab):
    """Masks of -inf and of the type's lowest value that leave few tokens or none; rows
    with NaN or +inf; scores that are not finite; every beam done."""
    dtype = getattr(torch, dtype)
    logits, scores = _inputs(4, 4, vocab, dtype, 5)
    for low in (-math.inf, torch.finfo(dtype).min):
        x = logits.clone()
        allowed = torch.zeros(x.shape, dtype=torch.bool, device="cuda")
        allowed[..., 7] = allowed[..., vocab - 1] = True
        allowed[1, 2] = False
        allowed[2] = False
        x[~allowed] = low
        _check(x, scores, 8)
    x = logits.clone()
    x[0, 1, 3] = math.nan
    x[1, 0, vocab - 1] = math.inf
    x[2, :, 0] = math.nan
    s = scores.clone()
    s[0, 0], s[0, 2], s[3, 0], s[3, 1] = -math.inf, math.inf, math.nan, -math.inf
    _check(x, s, 12)
    _check(x, torch.full_like(s, -math.inf), 12)
    done = torch.zeros((4, 4), dtype=torch.bool, device="cuda")
    done[0] = done[2, 1] = done[3, 1] = True
    _check(x, s, 12, done, 2)
    # the first step: all beams alike, one of them live
    first = torch.full((4, 4), -math.inf, device="cuda")
    first[:, 0] = 0
    _check(logits[:, :1].expand(4, 4, vocab), first, 8)


@pytest.mark.parametrize("dtype", ["float32", "bfloat16", "float16"])
@pytest.mark.parametrize("groups,beams,vocab,count", [(8, 64, 9001, 8), (8, 64, 16384, 20), (22, 16, 16390, 11)])
def test_large_grids(dtype, groups, beams, vocab, count):
    """Many rows and long lists: plain rows, ties, masks, NaN, done beams, rising rows."""
    dtype = getattr(torch, dtype)
    logits, scores = _inputs(groups, beams, vocab, dtype, vocab)
    low = torch.finfo(dtype).min
    logits[1] = 0                                        # more ties than any list holds
    logits[2, :, :vocab - 3] = -math.inf
    logits[3, :, :vocab - 3] = low
    logits[3, 1] = low
    logits[4, 1, 5], logits[4, 2, vocab - 1], logits[4, 3] = math.nan, math.inf, -math.inf
    logits[5] = torch.linspace(-20, 20, vocab, device="cuda").to(dtype)
    logits[6] = torch.linspace(20, -20, vocab, device="cuda").to(dtype)
    logits[7] = torch.randint(0, 3, (beams, vocab), generator=torch.Generator().manual_seed(7)).cuda().to(dtype)
    scores[1] = scores[7] = 0
    scores[4, 0], scores[4, 4] = -math.inf, math.nan
    _check(logits, scores, count)
    done = torch.rand((groups, beams), generator=torch.Generator().manual_seed(count)).cuda() < 0.3
    _check(logits, scores, count, done, 2)


@pytest.mark.parametrize("order", ["rising", "falling"])
@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
def test_sorted_rows(order, dtype):
    """The best tokens adjacent, at either end."""
    x = torch.linspace(-20, 20, 20000, device="cuda")
    x = (x if order == "rising" else x.flip(0)).to(getattr(torch, dtype))
    _check(x.expand(2, 3, 20000).contiguous(), torch.tensor([[0., -1, -2], [-3, 0, -.5]], device="cuda"), 64)


def test_strided_rows():
    """A padded vocabulary, one position of a sequence's logits, and odd offsets."""
    gen = torch.Generator().manual_seed(2)
    for dtype in (torch.float32, torch.bfloat16):
        wide = torch.randn((2, 3, 5, 4096), generator=gen).cuda().to(dtype)
        scores = torch.rand((2, 3), generator=gen).cuda()
        _check(wide[:, :, -1, :4001], scores, 8)
        _check(wide[:, :, 2, 3:4000], scores, 8)
        _check(wide[:, :, 2, ::2], scores, 8)
        _check(wide[..., 0, :].transpose(0, 1), scores.t(), 5)


def test_close_scores_of_beams():
    """Two beams a few float32 steps apart: 64 bits tell them apart."""
    gen = torch.Generator().manual_seed(9)
    row = torch.randn((1, 1, 6000), generator=gen).cuda()
    logits = row.expand(8, 2, 6000).contiguous()
    scores = torch.full((8, 2), -17.25, device="cuda")
    for g in range(8):
        scores[g, g % 2] = torch.nextafter(scores[g, g % 2], torch.tensor(0.0, device="cuda"))
    _check(logits, scores, 16)


def test_replay():
    from pkv import ops

    logits, scores = _inputs(3, 4, 9999, torch.bfloat16)
    ops.beam_select(logits, scores, 8)
    graph, stream = torch.cuda.CUDAGraph(), torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream), torch.cuda.graph(graph, stream=stream):
        got = ops.beam_select(logits, scores, 8)
    torch.cuda.current_stream().wait_stream(stream)
    for k in range(4):
        x, s = _inputs(3, 4, 9999, torch.bfloat16, 20 + k)
        logits.copy_(x)
        scores.copy_(s)
        graph.replay()
        want = ops.beam_select(logits, scores, 8)
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_masks_that_leave_lanes_without_tokens():
    """Many tokens from rows where most lanes of a wave hold none, and scattered ones."""
    gen = torch.Generator().manual_seed(3)
    for dtype in (torch.float32, torch.bfloat16):
        x = torch.randn((2, 3, 30000), generator=gen).cuda().to(dtype)
        scores = torch.rand((2, 3), generator=gen).cuda()
        for share in (0.001, 0.03, 0.5):
            y = x.clone()
            y[(torch.rand(x.shape, generator=gen) > share).cuda()] = -math.inf
            _check(y, scores, 64)
        z = torch.full_like(x, -math.inf)
        z[..., 4000:4100] = x[..., 4000:4100]
        _check(z, scores, 50)


def test_groups_with_more_candidates_than_lds_holds():
    """Equal values across many beams: more reach the bound than are ranked at once."""
    logits = torch.zeros((1, 64, 20000), device="cuda", dtype=torch.bfloat16)
    _check(logits, torch.zeros((1, 64), device="cuda"), 64)
    logits[0, 5, 19999] = 1
    _check(logits, torch.zeros((1, 64), device="cuda"), 64)
