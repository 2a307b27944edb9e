"""GPU: which tokens eviction keeps, against a plain selection, and their move to other
pages, bit for bit in the reference's page tensors."""

from __future__ import annotations

import numpy as np
import pytest

from cache_ops_case import filled

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")


@pytest.fixture(scope="module", autouse=True)
def _gpu():
    if not torch.cuda.is_available():
        pytest.skip("no GPU")


def _plain(mass, length, keep, sinks, recent):
    """Kept indices of one row (numpy float32)."""
    n = min(length, keep)
    r = min(recent, n)
    s = min(sinks, n - r)
    middle = list(range(s, length - r)) if n else []
    def rank(t):
        m = mass[t]
        return (0, 0.0, t) if np.isnan(m) else (1, -float(m), t)
    best = sorted(middle, key=rank)[:n - r - s]
    return sorted(list(range(s)) + best + list(range(length - r, length))) if n else []


def _check(mass, lens, keep, sinks, recent, **kw):
    from pkv import ops

    m = torch.from_numpy(mass).cuda()
    per = [keep] * len(lens) if isinstance(keep, int) else list(keep)
    kept, n, sums = ops.evict_select(m, lens, keep, sinks=sinks, recent=recent, with_mass=True, **kw)
    host, sums = kept.cpu().numpy(), sums.cpu().numpy()
    assert n.tolist() == [min(l, k) for l, k in zip(lens, per)]
    flat = mass.reshape(-1, *mass.shape[-3:])
    for layer in range(flat.shape[0]):
        for b, length in enumerate(lens):
            for h in range(mass.shape[-2]):
                want = _plain(flat[layer, b, h], length, per[b], sinks, recent)
                row = host.reshape(flat.shape[0], *host.shape[-3:])[layer, b, h]
                assert row[:len(want)].tolist() == want, (layer, b, h)
                assert (row[len(want):] == -1).all()
                got = sums.reshape(flat.shape[0], *sums.shape[-3:])[layer, b, h]
                assert got[:len(want)].tobytes() == flat[layer, b, h][want].tobytes()
                assert not got[len(want):].any()


@pytest.mark.parametrize("width", [1, 63, 64, 500, 1024, 4097, 9000])
@pytest.mark.parametrize("kind", ["spread", "few values", "all equal", "narrow"])
def test_select(width, kind):
    rng = np.random.default_rng(width)
    shape = (2, 3, 2, width)
    mass = {"spread": lambda: (rng.exponential(1.0, shape) ** 4), "few values": lambda: rng.integers(0, 3, shape),
            "all equal": lambda: np.full(shape, 0.25), "narrow": lambda: 1 + rng.random(shape) * 1e-5,
            }[kind]().astype(np.float32)
    lens = [width, max(1, width // 3), 0]
    for keep, sinks, recent in ((width, 4, 4), (width // 2, 4, 64), (1, 0, 0), (max(1, width // 7), 0, 3),
                                (0, 4, 4), (width + 9, 1, 1), (max(1, width - 1), 2, 5)):
        _check(mass, lens, keep, sinks, recent)
    _check(mass[0], lens, 10, 4, 5)


def test_select_unusual_sums():
    """Infinities, NaN of either sign, the type's extremes, zeros of either sign, denormals."""
    rng = np.random.default_rng(3)
    values = np.array([np.inf, -np.inf, np.nan, -np.nan, 0.0, -0.0, 1e-45, -1e-45, 3.4028235e38, -3.4028235e38, 1.0,
                       1.0000001], np.float32)
    mass = values[rng.integers(0, len(values), (1, 2, 2, 700))]
    mass[0, 1, 1] = np.nan
    for keep in (1, 60, 300, 640, 699):
        _check(mass, [700, 650], keep, 3, 11)


def test_select_budgets_rows_and_garbage_past_the_length():
    from pkv import ops

    rng = np.random.default_rng(4)
    mass = rng.random((2, 6, 3, 300)).astype(np.float32)
    mass[..., 200:] = np.nan                       # past every length
    m = torch.from_numpy(mass).cuda()
    lens, rows, keep = [200, 150, 9, 77], [5, 0, 3, 9], [50, 200, 0, 10]   # row 9 does not exist
    kept, n, sums = ops.evict_select(m, lens, torch.tensor(keep), max_keep=64, sinks=2, recent=5, rows=rows,
                                     with_mass=True)
    assert n.tolist() == [50, 64, 0, 0]
    assert sums.shape == (2, 6, 3, 64)
    for layer in range(2):
        for b in range(3):
            for h in range(3):
                want = _plain(mass[layer, rows[b], h], lens[b], min(keep[b], 64), 2, 5)
                assert kept[layer, b, h].tolist() == want + [-1] * (64 - len(want))
                assert sums[layer, rows[b], h, :len(want)].cpu().numpy().tobytes() == \
                    mass[layer, rows[b], h][want].tobytes()
    assert (kept[:, 3] == -1).all() and not sums[:, [1, 2, 4]].any()
    # in place: the kept sums at the front, zeros to max_keep, the rest as it was
    ops.evict_select(m, lens, torch.tensor(keep), max_keep=64, sinks=2, recent=5, rows=rows, new_mass=m)
    after = m.cpu().numpy()
    assert after[:, rows[:3], :, :64].tobytes() == sums[:, rows[:3]].cpu().numpy().tobytes()
    assert after[..., 64:].tobytes() == mass[..., 64:].tobytes()
    assert after[:, [1, 2, 4]].tobytes() == mass[:, [1, 2, 4]].tobytes()


@pytest.mark.parametrize("length,keep", [(16384, 4000), (16385, 16000), (32768, 9), (40000, 1000), (70001, 69000), (131072, 65536)])
def test_select_long(length, keep):
    rng = np.random.default_rng(length)
    mass = (rng.exponential(1.0, (1, 1, 2, length)) ** 3).astype(np.float32)
    mass[0, 0, 1] = np.round(mass[0, 0, 1], 1)
    _check(mass, [length], keep, 4, 100)


def test_select_in_place_long():
    from pkv import ops

    rng = np.random.default_rng(8)
    m = torch.from_numpy(rng.random((2, 2, 40000), dtype=np.float32)).cuda()
    kept, _, apart = ops.evict_select(m, [40000, 35000], 30000, recent=10, with_mass=True)
    again, _, _ = ops.evict_select(m, [40000, 35000], 30000, recent=10, new_mass=m)
    assert torch.equal(kept, again) and torch.equal(m[..., :30000], apart)


@pytest.mark.parametrize("length", [300, 3000, 16384, 16385, 40000])
def test_select_protected_tokens_beside_nan(length):
    """NaN sums come before numbers and after protected tokens, in place as well."""
    from pkv import ops

    rng = np.random.default_rng(length)
    mass = rng.random((1, 1, 2, length), dtype=np.float32)
    mass[0, 0, 0, rng.permutation(length)[:length // 3]] = np.nan
    mass[0, 0, 1] = np.nan
    for keep, sinks, recent in ((50, 20, 30), (51, 20, 30), (length // 4, 4, 60), (length - 1, 4, 60)):
        _check(mass, [length], keep, sinks, recent)
        m = torch.from_numpy(mass).cuda()
        _, _, apart = ops.evict_select(m, [length], keep, sinks=sinks, recent=recent, with_mass=True)
        ops.evict_select(m, [length], keep, sinks=sinks, recent=recent, new_mass=m)
        assert torch.equal(m[..., :keep].view(torch.int32), apart.view(torch.int32))


# ---- pages --------------------------------------------------------------------------------


def _tokens(fmt, pool, ids):
    """Reference page tensors of pages ``ids`` by token: each [HK, tokens, ...] as bytes."""
    from pkv import ops

    parts = ops.gather_pages(fmt, pool, torch.as_tensor(ids, dtype=torch.int32, device="cuda"))
    return [p.cpu().view(torch.uint8).transpose(0, 1).flatten(1, 2).numpy() for p in parts]


def _move(fmt, lens, kept, new_lens, *, layers=1, spoil=None):
    from pkv import ops

    p = fmt.page_tokens
    most = kept.shape[-1]
    dst_pages = max(1, -(-most // p))
    pools, table, spare = [], None, None
    for l in range(layers):
        pool, table, spare = filled(fmt, lens, seed=1, extra_pages=dst_pages * len(lens), junk=0x35 + l)
        pools.append(pool)
    dst = torch.from_numpy(spare.reshape(len(lens), dst_pages).copy()).cuda()
    if spoil:
        spoil(table, dst)
    before = [x.clone() for x in pools]
    kept_d = torch.from_numpy(kept).cuda()
    ops.evict_pages(fmt, pools if layers > 1 else pools[0], kept_d, new_lens, table, dst)
    for l in range(layers):
        written = set()
        for b in range(len(lens)):
            ids = dst[b].cpu().numpy()
            ok = (ids >= 0) & (ids < pools[l].shape[0])
            got = _tokens(fmt, pools[l], np.where(ok, ids, 0))
            held = _tokens(fmt, before[l], np.where(ok, ids, 0))
            src_ids = table[b].cpu().numpy()
            src_ok = (src_ids >= 0) & (src_ids < pools[l].shape[0])
            src = _tokens(fmt, before[l], np.where(src_ok, src_ids, 0))
            written |= set(ids[ok].tolist())
            k = kept.reshape(layers, len(lens), fmt.num_kv_heads, most)[l, b]
            for x, y, z in zip(got, held, src):
                want = y.copy()
                for h in range(fmt.num_kv_heads):
                    for i in range(min(int(new_lens[b]), most)):
                        t = int(k[h, i])
                        if 0 <= t < len(src_ok) * p and src_ok[t // p] and ok[i // p]:
                            want[h, i] = z[h, t]
                for i in range(len(ids)):
                    if ok[i]:
                        assert np.array_equal(x[:, i * p:(i + 1) * p], want[:, i * p:(i + 1) * p]), (l, b, i)
        rest = [i for i in range(pools[l].shape[0]) if i not in written]
        assert torch.equal(pools[l][rest], before[l][rest])


def _kept(rng, lens, hk, most, layers=1):
    kept = np.full((layers, len(lens), hk, most), -1, np.int32)
    new = [min(n, most) for n in lens]
    for l in range(layers):
        for b, n in enumerate(lens):
            for h in range(hk):
                kept[l, b, h, :new[b]] = np.sort(rng.permutation(n)[:new[b]])
    return (kept if layers > 1 else kept[0]), new


@pytest.mark.parametrize("bits,dim,group", [(8, 64, 32), (8, 128, 64), (8, 256, 128), (4, 64, 64), (4, 128, 32),
                                            (4, 256, 64), (16, 64, 32), (16, 128, 32), (16, 256, 32), (8, 80, 32),
                                            (4, 37, 32), (16, 100, 32)])
@pytest.mark.parametrize("page", [16, 64])
def test_pages(bits, dim, group, page):
    from pkv import ops

    fmt = ops.PageFormat(2, dim, page, bits, group, torch.bfloat16 if dim != 128 else torch.float16)
    rng = np.random.default_rng(dim + page)
    for most in (1, 15, 16, 17, 61, 130):
        lens = [200, 90, 5, 0]
        kept, new = _kept(rng, lens, 2, most)
        _move(fmt, lens, kept, new)


@pytest.mark.parametrize("bits", [4, 8, 16])
def test_pages_of_layers_and_unmapped_ones(bits):
    from pkv import ops

    fmt = ops.PageFormat(3, 128, 32, bits, 64, torch.bfloat16)
    rng = np.random.default_rng(bits)
    lens = [150, 100]
    kept, new = _kept(rng, lens, 3, 70, layers=3)
    _move(fmt, lens, kept, new, layers=3)

    def spoil(table, dst):
        table[0, 1] = -1          # a source page that is not mapped
        table[1, 0] = 1 << 20     # ... and one that does not exist
        dst[0, 2] = -1
        dst[1, 1] = 1 << 20

    kept[:, 1, :, 3] = -1
    kept[:, 1, :, 5] = 1 << 28
    _move(fmt, lens, kept, [70, 33], layers=3, spoil=spoil)


def test_select_and_pages_replay():
    """Selection and move as one graph, replayed over other sums, against eager calls."""
    from pkv import ops

    fmt = ops.PageFormat(2, 128, 16, 8, 64, torch.bfloat16)
    lens = torch.tensor([300, 120], dtype=torch.int32, device="cuda")
    pool, table, spare = filled(fmt, lens.tolist(), extra_pages=20)
    other = pool.clone()
    dst = torch.from_numpy(spare.reshape(2, 10).copy()).cuda()
    mass = torch.rand((2, 2, table.shape[1] * 16), device="cuda")

    def step(to):
        kept, n, sums = ops.evict_select(mass, lens, 150, sinks=4, recent=16, with_mass=True)
        ops.evict_pages(fmt, to, kept, n, table, dst)
        return kept, n, sums

    step(pool)
    graph, stream = torch.cuda.CUDAGraph(), torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream), torch.cuda.graph(graph, stream=stream):
        got = step(pool)
    torch.cuda.current_stream().wait_stream(stream)
    for k in range(4):
        mass.copy_(torch.rand(mass.shape, device="cuda"))
        lens.copy_(torch.tensor([300 - 31 * k, 120]))
        graph.replay()
        want = step(other)
        torch.cuda.synchronize()
        assert all(torch.equal(x, y) for x, y in zip(got, want))
        assert torch.equal(pool, other)
