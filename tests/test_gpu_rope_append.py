"""GPU: rotation with append against the rotation in 64 bits and, bit for bit, against the
append of the k and v that come out."""

from __future__ import annotations

import numpy as np
import pytest

from step_case import assert_turned, turned64

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")


@pytest.fixture(scope="module", autouse=True)
def _gpu():
    if not torch.cuda.is_available():
        pytest.skip("no GPU")


def _inv_freq(half, theta=10000.0):
    return (theta ** (-torch.arange(half, dtype=torch.float64) / max(half, 1))).float()


def _check(bits, dim, group=32, *, page=16, kv_heads=2, heads=6, dtype=torch.bfloat16, lens=(1, 1, 1), cached=None,
           half=None, axes=0, padded=False, spare=0, offset=0, unmap=(), positions=None, inv_freq=None, edit=None,
           behind=0):
    from pkv import ops

    fmt = ops.PageFormat(kv_heads, dim, page, bits, group, dtype)
    gen = torch.Generator().manual_seed(dim * 31 + len(lens))
    batch, half = len(lens), dim // 2 if half is None else half
    cached = [(7 * b + 3) % 40 for b in range(batch)] if cached is None else cached
    width = (heads + 2 * kv_heads) * dim
    tokens = max(lens) + 2 if padded else 0
    rows = batch * tokens if padded else sum(lens) + behind
    store = torch.randn((rows, width + spare), generator=gen).to(dtype).cuda()
    flat = torch.empty(store.numel() + offset, dtype=dtype, device="cuda")
    flat[offset:] = store.flatten()
    qkv = flat[offset:].view(rows, width + spare)[:, :width]
    if edit:
        edit(qkv)
    starts = np.concatenate([[0], np.cumsum(lens)])
    counts = [-(-(max(c, 0) + n) // page) for c, n in zip(cached, lens)]
    ids = np.random.default_rng(3).permutation(sum(counts) + 2).astype(np.int32)
    table = np.full((batch, max(max(counts), 1)), -1, np.int32)
    at = 0
    for b, n in enumerate(counts):
        table[b, :n] = ids[at:at + n]
        at += n
    for b, p in unmap:
        table[b, p] = -1
    pool = torch.randint(0, 256, (len(ids), fmt.page_bytes), generator=gen, dtype=torch.uint8).cuda()
    before = pool.clone()
    inv = _inv_freq(half) if inv_freq is None else inv_freq
    lead = (batch, tokens) if padded else (rows,)
    place = np.zeros((max(axes, 1),) + lead, np.int64)
    live = np.zeros(lead, bool)
    for b, n in enumerate(lens):
        at = (b, slice(0, n)) if padded else slice(starts[b], starts[b] + n)
        place[(slice(None),) + (at if padded else (at,))] = cached[b] + np.arange(n)
        live[at] = True
    kw = {}
    if axes:
        place += np.random.default_rng(5).integers(0, 300, place.shape)
        kw["axes"] = torch.from_numpy(np.arange(half) * axes // max(half, 1)).int().cuda()
        kw["positions"] = torch.from_numpy(place.astype(np.int32)).cuda()
    elif positions is not None:
        place[0][live] = positions
        kw["positions"] = torch.from_numpy(place[0].astype(np.int32)).cuda()
    x = qkv.view(batch, tokens, width) if padded else qkv
    if padded:
        kw["widths"] = torch.tensor(lens, dtype=torch.int32, device="cuda")
    else:
        kw["row_starts"] = torch.from_numpy(starts.astype(np.int32)).cuda()
    shapes = [(batch, n, tokens, dim) if padded else (rows, n, dim) for n in (heads, kv_heads, kv_heads)]
    out = [torch.full(s, 77.0, dtype=dtype, device="cuda") for s in shapes]
    got = ops.rope_append(fmt, pool, x, torch.from_numpy(table).cuda(), cached, inv.cuda(), heads, with_kv=True,
                          out=out, **kw)
    assert all(g is o for g, o in zip(got, out))
    alone = pool.clone()
    q = ops.rope_append(fmt, alone, x, torch.from_numpy(table).cuda(), cached, inv.cuda(), heads, **kw)
    q, k, v = [(t.transpose(1, 2) if padded else t) for t in (q, *got[1:])]
    assert torch.equal(alone, pool)
    mask = torch.from_numpy(live).cuda()
    first = out[0].transpose(1, 2) if padded else out[0]
    assert torch.equal(q[mask].view(torch.int16), first[mask].view(torch.int16))
    for t in (first, k, v):
        assert bool((t[~mask] == 77.0).all())       # rows of no sequence
    # the rotation
    axis = np.arange(half) * max(axes, 1) // max(half, 1)
    angles = np.moveaxis(place[axis], 0, -1).astype(np.float64) * inv.double().numpy()
    source = qkv.double().cpu().numpy().reshape(lead + (heads + 2 * kv_heads, dim))
    want, size = turned64(source[live], angles[live], half)
    if edit is None:
        assert_turned(first[mask], want[:, :heads], size[:, :heads], dtype)
        assert_turned(k[mask], want[:, heads:heads + kv_heads], size[:, heads:heads + kv_heads], dtype)
    source = qkv.reshape(lead + (heads + 2 * kv_heads, dim))[..., heads + kv_heads:, :]
    assert torch.equal(v[mask].view(torch.int16), source[mask].view(torch.int16))
    # the pages: what the append makes of k and v
    n = max(max(lens), 1)
    sides = torch.zeros((2, batch, kv_heads, n, dim), dtype=dtype, device="cuda")
    for b, w in enumerate(lens):
        at = (b, slice(0, w)) if padded else slice(starts[b], starts[b] + w)
        for i, t in enumerate((k, v)):
            sides[i, b, :, :w] = t[at].transpose(0, 1)
    widths = torch.tensor([w if c >= 0 else 0 for w, c in zip(lens, cached)], dtype=torch.int32, device="cuda")
    ops.append_quantize(fmt, before, sides[0], sides[1], torch.from_numpy(table).cuda(), cached, widths)
    assert torch.equal(before, pool)


LAYOUTS = [(8, 64, 32), (8, 64, 64), (8, 128, 32), (8, 128, 64), (8, 128, 128), (8, 256, 64), (4, 64, 32),
           (4, 128, 64), (4, 128, 128), (4, 256, 32), (4, 256, 128), (16, 64, 32), (16, 128, 32), (16, 256, 32),
           (8, 80, 32), (4, 96, 32), (4, 37, 32), (16, 100, 32), (16, 7, 32), (8, 2, 32), (8, 1, 32)]


@pytest.mark.parametrize("dtype", ["bfloat16", "float16"])
@pytest.mark.parametrize("bits,dim,group", LAYOUTS)
@pytest.mark.parametrize("lens", [(1, 1, 1, 1, 1), (5, 0, 1, 3), (40, 0, 17, 1, 16, 130)])
def test_layouts(bits, dim, group, dtype, lens):
    _check(bits, dim, group, dtype=getattr(torch, dtype), lens=lens)


@pytest.mark.parametrize("bits", [4, 8, 16])
@pytest.mark.parametrize("page", [16, 32, 64, 128])
@pytest.mark.parametrize("lens,cached", [((1,), (0,)), ((1,), (5000,)), ((300, 1, 77), (0, 127, 129)),
                                         ((16, 32), (16, 0)), ((15, 33, 100), (15, 1, 31))])
def test_pages_and_starts(bits, page, lens, cached):
    _check(bits, 128, 64, page=page, lens=lens, cached=list(cached), heads=4, kv_heads=1)


@pytest.mark.parametrize("bits", [4, 8, 16])
@pytest.mark.parametrize("lens", [(1, 3, 2), (30, 0, 17), (70, 0, 47)])
def test_padded(bits, lens):
    _check(bits, 128, 64, lens=lens, padded=True)
    _check(bits, 64, 32, lens=lens, padded=True, axes=3, dtype=torch.float16)


@pytest.mark.parametrize("dim,half", [(128, 32), (128, 0), (128, 20), (80, 16), (256, 128), (64, 24)])
@pytest.mark.parametrize("lens", [(1, 2), (50, 20), (110, 45)])
def test_part_of_a_head_and_axes(dim, half, lens):
    _check(8, dim, 32, lens=lens, half=half)
    _check(16, dim, 32, lens=lens, half=half, axes=3)
    _check(4, dim, 32, lens=lens, half=half, axes=2, kv_heads=1, heads=1)


@pytest.mark.parametrize("spare,offset", [(8, 0), (24, 8), (3, 0), (0, 1), (8, 4)])
@pytest.mark.parametrize("lens", [(1, 1), (33, 50), (77, 90)])
def test_strided_rows(spare, offset, lens):
    _check(8, 128, 64, lens=lens, spare=spare, offset=offset)


@pytest.mark.parametrize("bits", [4, 16])
@pytest.mark.parametrize("lens", [(2, 1, 3), (70, 20, 33), (70, 50, 33)])
def test_places_without_a_page(bits, lens):
    """Unmapped pages, a sequence that is not one, rows behind the last sequence."""
    _check(bits, 128, 64, lens=lens, cached=[30, 0, 14], unmap=[(0, 1), (1, 0)], behind=5)


@pytest.mark.parametrize("lens", [(1, 1, 2), (64, 9, 40), (90, 9, 70)])
def test_far_positions(lens):
    """Angles whose 32-bit product would have no digit left, and frequencies above one."""
    n = sum(lens)
    far = np.random.default_rng(1).integers(0, 2 ** 31 - 1, n)
    far[:3] = [2 ** 31 - 1, 0, 131072]
    _check(8, 128, 64, lens=lens, positions=far)
    _check(16, 64, 32, lens=lens, positions=-(far // 2))
    _check(8, 64, 32, lens=lens, positions=far // 1000, inv_freq=torch.linspace(0, 40, 32))


@pytest.mark.parametrize("bits", [4, 8, 16])
@pytest.mark.parametrize("lens", [(1, 2, 1), (40, 17, 3), (98, 47, 3)])
def test_values_that_are_not_finite(bits, lens):
    def edit(qkv):
        qkv[0, 5], qkv[1, -3], qkv[2, 700], qkv[3, -130] = float("inf"), float("nan"), -float("inf"), 60000.0
        qkv[2, 701] = float("nan")

    for dtype in (torch.bfloat16, torch.float16):
        _check(bits, 128, 64, lens=lens, edit=edit, dtype=dtype)


def test_negative_start():
    """A sequence that starts before its cache has no rows."""
    from pkv import ops

    for n in (1, 20, 64):
        fmt = ops.PageFormat(2, 64, 16, 8, 32, torch.bfloat16)
        pool = ops.allocate_pool(fmt, 8)
        qkv = torch.randn((2 * n, 6 * 64), device="cuda").bfloat16()
        out = torch.full((2 * n, 2, 64), 7.0, dtype=torch.bfloat16, device="cuda")
        table = torch.arange(8, dtype=torch.int32, device="cuda").view(2, 4)
        ops.rope_append(fmt, pool, qkv, table, [-3, 0], _inv_freq(32).cuda(), 2, row_starts=[0, n, 2 * n], out=out)
        assert bool((out[:n] == 7.0).all()) and not bool((out[n:] == 7.0).all())
        assert int(pool[:4].count_nonzero()) == 0 and int(pool[4:].count_nonzero()) > 0


def test_refusals():
    from pkv import ops

    fmt = ops.PageFormat(2, 64, 16, 8, 32, torch.bfloat16)
    pool = ops.allocate_pool(fmt, 8)
    qkv = torch.zeros((4, 6 * 64), dtype=torch.bfloat16, device="cuda")
    table = torch.zeros((2, 4), dtype=torch.int32, device="cuda")
    inv = _inv_freq(32).cuda()
    good = dict(row_starts=[0, 2, 4])

    def call(pool=pool, qkv=qkv, table=table, start=(0, 0), inv=inv, heads=2, **kw):
        return ops.rope_append(fmt, pool, qkv, table, list(start), inv, heads, **{**good, **kw})

    call()
    row = torch.zeros(4, dtype=torch.int32, device="cuda")
    for bad in (dict(qkv=qkv.half()), dict(qkv=qkv.cpu()), dict(heads=3), dict(heads=0), dict(row_starts=[0, 4]),
                dict(row_starts=None), dict(widths=[1, 1]), dict(start=(0,)), dict(table=table[:1]),
                dict(inv=inv.double()), dict(inv=_inv_freq(33).cuda()), dict(positions=row[:3]), dict(axes=row),
                dict(positions=row, axes=torch.zeros(31, dtype=torch.int32)), dict(pool=pool[:, :64].contiguous()),
                dict(positions=torch.zeros((9, 4), dtype=torch.int32), axes=torch.zeros(32, dtype=torch.int32)),
                dict(out=torch.zeros((4, 2, 64), device="cuda")),
                dict(out=[torch.zeros((4, 2, 64), dtype=torch.bfloat16, device="cuda")] * 2, with_kv=True)):
        with pytest.raises(ValueError):
            call(**bad)
