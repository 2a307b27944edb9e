"""GPU: causal attention within packed sequences against the same in 64 bits."""

from __future__ import annotations

import numpy as np
import pytest

from step_case import attention64, attention_bound, half_step

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")


@pytest.fixture(scope="module", autouse=True)
def _gpu():
    if not torch.cuda.is_available():
        pytest.skip("no GPU")


def _rows(lens, heads, kv_heads, dim, dtype, seed=0, gain=1.0, behind=0):
    gen = torch.Generator().manual_seed(seed + 17 * dim)
    total = sum(lens) + behind
    q, k, v = (torch.randn((total, n, dim), generator=gen) for n in (heads, kv_heads, kv_heads))
    starts = torch.from_numpy(np.concatenate([[0], np.cumsum(lens)]).astype(np.int32)).cuda()
    return [t.to(dtype).cuda() for t in (q * gain, k, v)], starts


def _compare(got, q, k, v, lens, scale, rows=None, skip=0):
    """Every row (or ``rows`` of every sequence) of packed sequences from row ``skip`` on."""
    gqa, dim = q.shape[1] // k.shape[1], q.shape[2]
    worst, at = 0.0, skip
    q64, k64, v64, got64 = (t.double().cpu().numpy() for t in (q, k, v, got))
    for n in lens:
        pick = np.arange(n) if rows is None else np.unique(np.clip(rows, 0, n - 1))
        for h in range(q.shape[1]):
            if n == 0:
                continue
            with np.errstate(invalid="ignore", over="ignore"):
                want, weight, terms = attention64(q64[at:at + n, h][pick], k64[at:at + n, h // gqa],
                                                  v64[at:at + n, h // gqa], pick + 1, scale)
            bound = attention_bound(want, weight, terms, scale, q.dtype, dim=dim, tokens=n, operand=half_step(q.dtype))
            off = np.abs(got64[at:at + n, h][pick] - want)
            assert np.all(off <= bound), (n, h, float(np.nanmax(off / bound)))
            worst = max(worst, float((off / bound).max()))
        at += n
    return worst


def _check(lens, heads=4, kv_heads=2, dim=64, dtype=torch.bfloat16, *, seed=0, gain=1.0, behind=0, rows=None):
    from pkv import ops

    (q, k, v), starts = _rows(lens, heads, kv_heads, dim, dtype, seed, gain, behind)
    scale = dim ** -0.5
    out = torch.full_like(q, 7.0)
    got = ops.prompt_attention(q, k, v, starts, scale=scale, out=out)
    assert got is out
    total = sum(lens)
    assert bool((out[total:] == 7.0).all())
    _compare(out, q, k, v, lens, scale, rows)
    alone = ops.prompt_attention(q, k, v, starts, scale=scale)
    assert torch.equal(alone[:total].view(torch.int16), out[:total].view(torch.int16))


@pytest.mark.parametrize("dtype", ["bfloat16", "float16"])
@pytest.mark.parametrize("dim", [8, 37, 64, 72, 80, 96, 128, 136, 192, 256])
@pytest.mark.parametrize("heads,kv_heads", [(4, 1), (6, 2), (3, 3), (7, 1), (16, 1)])
def test_layouts(dim, dtype, heads, kv_heads):
    _check([1, 40, 0, 97, 33], heads, kv_heads, dim, getattr(torch, dtype), behind=3)


@pytest.mark.parametrize("n", [1, 2, 31, 32, 33, 63, 64, 65, 127, 128, 129, 255, 256, 257, 300, 511, 513])
@pytest.mark.parametrize("heads,kv_heads,dim", [(1, 1, 128), (4, 1, 128), (2, 1, 256)])
def test_lengths(n, heads, kv_heads, dim):
    _check([n], heads, kv_heads, dim)
    _check([n, 1, n + 1, 0, 3], heads, kv_heads, dim, torch.float16)


@pytest.mark.parametrize("heads,kv_heads,dim,lens", [
    (32, 8, 128, [1500, 700, 33]), (32, 8, 64, [900, 1, 2100]), (28, 4, 128, [2500]), (16, 16, 128, [1100, 1300]),
    (64, 8, 96, [1000, 40])])
def test_large(heads, kv_heads, dim, lens):
    """Grids of the widest form, some of the rows."""
    rows = np.concatenate([np.arange(3), [31, 32, 63, 64, 65, 500, 511, 512, 1023, 1300, 1400], np.arange(2090, 2500, 37),
                           [699, 698, 1499, 899, 2099, 2499]])
    _check(lens, heads, kv_heads, dim, rows=rows)


@pytest.mark.parametrize("batch", [2, 3, 4, 7, 12, 13, 64, 70])
@pytest.mark.parametrize("heads,kv_heads", [(4, 1), (6, 2)])
def test_orders(batch, heads, kv_heads):
    """Sequences of unlike lengths, empty ones among them, as blocks are found in each order."""
    rng = np.random.default_rng(batch)
    lens = [int(n) for n in rng.integers(0, 200, batch)]
    lens[0], lens[-1], lens[batch // 2] = 300, 33, 0
    _check(lens, heads, kv_heads, behind=3)


def test_many_sequences():
    rng = np.random.default_rng(0)
    _check([int(n) for n in rng.integers(0, 40, 150)], 2, 1, 64)
    _check([int(n) for n in rng.integers(1, 300, 64)], 4, 1, 128, rows=np.array([0, 1, 31, 32, 100, 250, 299]))
    _check([int(n) for n in rng.integers(1, 300, 65)], 4, 1, 128, rows=np.array([0, 1, 31, 32, 100, 250, 299]))


@pytest.mark.parametrize("gain", [30.0, 1e-6, 300.0])
@pytest.mark.parametrize("dtype", ["bfloat16", "float16"])
def test_sharp_and_flat_weights(gain, dtype):
    _check([70, 400], 4, 2, 128, getattr(torch, dtype), gain=gain)


def test_rising_and_falling_scores():
    """The running maximum moves at every tile, or never again."""
    from pkv import ops

    for sign in (1.0, -1.0):
        (q, k, v), starts = _rows([700], 4, 1, 128, torch.float16)
        k[:, 0, 0] = sign * torch.arange(700).cuda() / 8
        q[..., 0] = 6.0
        got = ops.prompt_attention(q, k, v, starts, scale=1.0)
        _compare(got, q, k, v, [700], 1.0)


@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("dtype", ["bfloat16", "float16"])
def test_later_rows_that_are_not_finite(dim, dtype):
    """Infinities and NaN in a later row, the next sequence's and rows of no sequence change
    nothing before them."""
    from pkv import ops

    dtype = getattr(torch, dtype)
    lens = [45, 130, 70]
    (q, k, v), starts = _rows(lens, 8, 2, dim, dtype, behind=4)
    clean = ops.prompt_attention(q, k, v, starts, scale=0.1)
    for bad in (float("nan"), float("inf"), -float("inf")):
        for at in ((45 + 100, 20), (45 + 129, 0), (44, 5), (45 + 128, dim - 1), (45 + 127, 7)):
            k2, v2 = k.clone(), v.clone()
            k2[at[0], 1, at[1]] = bad
            v2[at[0], :, at[1]] = bad
            v2[-4:], k2[-4:] = bad, bad
            got = ops.prompt_attention(q, k2, v2, starts, scale=0.1)
            first, seq = at[0], int(at[0] >= 45)
            end = [45, 175][seq]
            keep = torch.ones(249, dtype=torch.bool)
            keep[first:end] = False
            keep[245:] = False
            assert torch.equal(got[keep].view(torch.int16), clean[keep].view(torch.int16))
            # rows that see it are not finite there
            assert not bool(torch.isfinite(got[first:end, :4, at[1]]).any())


@pytest.mark.parametrize("dim", [64, 128, 256])
def test_queries_that_are_not_numbers(dim):
    """A query with a NaN has a NaN result, in its row and head alone."""
    from pkv import ops

    gen = torch.Generator().manual_seed(dim)
    q, k, v = (torch.randn((300, h, dim), generator=gen).cuda().bfloat16() for h in (4, 2, 2))
    starts = [0, 100, 300]
    want = ops.prompt_attention(q, k, v, starts, scale=0.1)
    rows = [(0, 1), (50, 0), (99, 3), (100, 2), (231, 1)]
    for at in rows:
        q[at][5] = float("nan")
    got = ops.prompt_attention(q, k, v, starts, scale=0.1)
    for at in rows:
        assert bool(got[at].isnan().all())
        got[at] = want[at]
    assert torch.equal(got, want)


def test_an_infinite_value_among_finite_ones():
    """A visible infinity gives itself, both signs NaN, with finite scores."""
    from pkv import ops

    (q, k, v), starts = _rows([64], 4, 1, 64, torch.bfloat16)
    v[40, 0, 3] = float("inf")
    v[50, 0, 3] = -float("inf")
    got = ops.prompt_attention(q, k, v, starts, scale=0.1)
    assert bool(torch.isfinite(got[:40]).all())
    assert bool((got[40:50, :, 3] == float("inf")).all())
    assert bool(got[50:, :, 3].isnan().all())
    assert bool(torch.isfinite(got[:, :, 4]).all())


@pytest.mark.parametrize("spare", [0, 8, 3])
def test_views_of_a_projection(spare):
    from pkv import ops

    lens, heads, kv_heads, dim = [50, 130], 4, 2, 64
    (q, k, v), starts = _rows(lens, heads, kv_heads, dim, torch.float16)
    width = (heads + 2 * kv_heads) * dim
    rows = torch.cat([t.flatten(1) for t in (q, k, v)] + [torch.zeros((180, spare), device="cuda").half()], 1)
    parts = rows[:, :width].unflatten(1, (-1, dim)).split((heads, kv_heads, kv_heads), 1)
    want = ops.prompt_attention(q, k, v, starts, scale=0.125)
    got = ops.prompt_attention(*parts, starts, scale=0.125)
    assert torch.equal(got, want)
    got = ops.prompt_attention(*(t.transpose(0, 1).contiguous().transpose(0, 1) for t in (q, k, v)), starts, scale=0.125)
    assert torch.equal(got, want)


def test_starts_that_leave_rows_out():
    """Rows before the first sequence and behind the last are not touched."""
    from pkv import ops

    (q, k, v), _ = _rows([100], 4, 2, 64, torch.bfloat16)
    out = torch.full_like(q, 3.0)
    ops.prompt_attention(q, k, v, [20, 50, 50, 90], scale=0.2, out=out)
    assert bool((out[:20] == 3.0).all()) and bool((out[90:] == 3.0).all())
    _compare(out, q, k, v, [30, 0, 40], 0.2, skip=20)


def test_refusals():
    from pkv import ops
    from pkv.modes import ModelCapabilityUnsupported

    (q, k, v), starts = _rows([10], 4, 2, 64, torch.bfloat16)
    for bad in ((q.float(), k, v), (q, k.half(), v), (q, k[:9], v), (q, k, v[:, :1]), (q[0], k, v), (q.cpu(), k, v),
                (q, k[..., :32], v[..., :32])):
        with pytest.raises(ValueError):
            ops.prompt_attention(*bad, starts, scale=1.0)
    for kw in (dict(scale=float("nan")), dict(scale=1.0, out=q[:, :2]), dict(scale=1.0, out=torch.zeros_like(q).float())):
        with pytest.raises(ValueError):
            ops.prompt_attention(q, k, v, starts, **kw)
    with pytest.raises(ValueError):
        ops.prompt_attention(q[:, :3].contiguous(), k, v, starts, scale=1.0)
    wide = torch.zeros((4, 1, 264), dtype=torch.bfloat16, device="cuda")
    with pytest.raises(ModelCapabilityUnsupported):
        ops.prompt_attention(wide, wide, wide, [0, 4], scale=1.0)
    assert ops.prompt_attention(q[:0], k[:0], v[:0], [0], scale=1.0).shape == (0, 4, 64)
