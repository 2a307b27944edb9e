"""GPU: the attention weight that a call's queries put on each cached token, against
the same in 64 bits over the pages' stored values."""

from __future__ import annotations

import numpy as np
import pytest

from cache_ops_case import filled, mass64, scale_of

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")


@pytest.fixture(scope="module", autouse=True)
def _gpu():
    if not torch.cuda.is_available():
        pytest.skip("no GPU")


def _format(bits, dim, group=32, page=16, hk=2, dtype=torch.bfloat16):
    from pkv import ops

    return ops.PageFormat(hk, dim, page, bits, group, dtype)


def _queries(fmt, batch, gqa, nq, seed=1, gain=1.0):
    gen = torch.Generator().manual_seed(seed)
    q = torch.randn((batch, fmt.num_kv_heads * gqa, nq, fmt.head_dim), generator=gen) * gain
    return q.cuda().to(fmt.dtype)


def _check(fmt, lens, gqa, nq, *, seed=0, gain=1.0, k_scale=1.0, q_pos=None, widths=None, unmap=(), **kw):
    from pkv import ops

    pool, table, _ = filled(fmt, lens, seed=seed, k_scale=k_scale)
    for b, page in unmap:
        table[b, page] = -1
    q = _queries(fmt, len(lens), gqa, nq, seed + 1, gain)
    scale = scale_of(fmt)
    want, bound = mass64(fmt, pool, table, lens, q, scale, q_pos=q_pos, widths=widths)
    rows = table.shape[0] + 2
    out = torch.full((rows, fmt.num_kv_heads, table.shape[1] * fmt.page_tokens), -7.0, device="cuda")
    place = list(range(rows))[::-1][:len(lens)]
    got = ops.attention_mass(fmt, pool, q, table, lens, scale=scale, q_pos=q_pos, widths=widths, out=out,
                             rows=place, **kw)
    assert got is out
    got = got.double().cpu().numpy()
    for b, n in enumerate(lens):
        n = min(n, out.shape[2])
        off = np.abs(got[place[b], :, :n] - want[b][:, :n])
        assert np.all(off <= bound[b][:, :n]), (b, float((off / bound[b][:, :n]).max()))
        assert np.all(got[place[b], :, n:] == -7.0)
    for r in set(range(rows)) - set(place):
        assert np.all(got[r] == -7.0)


@pytest.mark.parametrize("dtype", ["bfloat16", "float16"])
@pytest.mark.parametrize("bits,dim,group", [
    (8, 64, 32), (8, 64, 64), (8, 128, 32), (8, 128, 64), (8, 128, 128), (8, 256, 32), (8, 256, 64), (8, 256, 128),
    (4, 64, 32), (4, 64, 64), (4, 128, 32), (4, 128, 64), (4, 128, 128), (4, 256, 32), (4, 256, 64), (4, 256, 128),
    (16, 64, 32), (16, 128, 32), (16, 256, 32), (8, 80, 32), (4, 37, 32), (16, 100, 32), (16, 7, 32), (8, 1, 32)])
@pytest.mark.parametrize("gqa,nq", [(4, 1), (8, 1), (1, 1), (2, 5), (3, 7), (4, 20)])
def test_layouts(bits, dim, group, dtype, gqa, nq):
    fmt = _format(bits, dim, group, 16, 2, getattr(torch, dtype))
    _check(fmt, [0, 1, 15, 17, 130, 333], gqa, nq)


@pytest.mark.parametrize("page", [16, 32, 64, 128])
@pytest.mark.parametrize("bits", [4, 8, 16])
@pytest.mark.parametrize("gqa,nq", [(4, 1), (2, 16)])
def test_pages_and_lengths(page, bits, gqa, nq):
    _check(_format(bits, 128, 64, page, 1), [1, 16, 31, 32, 33, 127, 128, 129, 511, 512, 513, 1025, 2500], gqa, nq)


@pytest.mark.parametrize("bits", [4, 8, 16])
@pytest.mark.parametrize("gqa,nq", [(8, 1), (2, 3), (4, 16), (1, 100)])
def test_rows_that_see_little(bits, gqa, nq):
    """Positions of any order, before the first token (nothing is seen), past the last;
    widths from none to all; a page that is not mapped, and a sequence without any."""
    fmt = _format(bits, 128, 64)
    lens = [5, 70, 300, 40, 0]
    rng = np.random.default_rng(nq)
    q_pos = np.stack([rng.integers(-3, max(n, 1) + 5, nq) for n in lens]).astype(np.int32)
    q_pos[3] = -1
    _check(fmt, lens, gqa, nq, q_pos=torch.from_numpy(q_pos).cuda(), unmap=[(2, 3), (1, 0), (2, 18)])
    _check(fmt, lens, gqa, nq, widths=[nq, 0, max(1, nq // 2), 1, nq], unmap=[(0, 0)])
    _check(fmt, lens, gqa, nq, q_pos=torch.from_numpy(q_pos).cuda(), widths=[nq, 1, nq - 1, nq, 0])


@pytest.mark.parametrize("bits", [4, 8, 16])
@pytest.mark.parametrize("gain,k_scale", [(30.0, 1.0), (1e4, 1e-4), (1e-6, 1.0), (3.0, 8.0)])
@pytest.mark.parametrize("gqa,nq", [(4, 1), (4, 8)])
def test_sharp_and_flat_weights(bits, gain, k_scale, gqa, nq):
    _check(_format(bits, 128, 64), [40, 700], gqa, nq, gain=gain, k_scale=k_scale)


@pytest.mark.parametrize("nq", [1, 24])
def test_sums_so_far(nq):
    """Accumulation in place and apart, with tokens that have no sum yet, and a mass
    narrower than the table."""
    from pkv import ops

    fmt = _format(8, 128, 64)
    lens = [100, 37, 5]
    pool, table, _ = filled(fmt, lens)
    q = _queries(fmt, 3, 4, nq)
    kw = dict(scale=scale_of(fmt))
    fresh = ops.attention_mass(fmt, pool, q, table, lens, **kw)
    assert fresh.shape == (3, 2, table.shape[1] * 16)
    old = torch.rand(fresh.shape, device="cuda")
    both = ops.attention_mass(fmt, pool, q, table, lens, mass=old, out=torch.zeros_like(old), **kw)
    counted = [90, 0, 7]
    old[1] = float("nan")          # sums that are not to be read
    old[0, :, 90:] = float("inf")
    kept = old.clone()
    got = ops.attention_mass(fmt, pool, q, table, lens, mass=old, counted=counted, **kw)
    assert got is old
    for b, n in enumerate(lens):
        c = min(counted[b], n)
        assert torch.equal(got[b, :, :c], kept[b, :, :c] + fresh[b, :, :c])
        assert torch.equal(got[b, :, c:n], fresh[b, :, c:n])
        assert torch.equal(got[b, :, n:].nan_to_num(), kept[b, :, n:].nan_to_num())
    assert torch.equal(both[0, :, :90], kept[0, :, :90] + fresh[0, :, :90])
    # a mass that ends inside the sequence: its tokens are all there are
    narrow = ops.attention_mass(fmt, pool, q, table, lens, out=torch.zeros((3, 2, 50), device="cuda"), **kw)
    pos = torch.tensor([[100 - nq + i for i in range(nq)], [37 - nq + i for i in range(nq)],
                        [5 - nq + i for i in range(nq)]], dtype=torch.int32, device="cuda")
    same = ops.attention_mass(fmt, pool, q, table, [50, 37, 5], q_pos=pos, **kw)
    assert torch.equal(narrow, same[..., :50])


def test_calls_are_deterministic_and_replay():
    """Two calls give the same bits; so does a captured call, replayed over other
    queries and lengths, beside eager calls."""
    from pkv import ops

    for bits, nq, gqa in ((8, 1, 4), (4, 16, 8), (16, 3, 2)):
        fmt = _format(bits, 128, 64)
        lens = torch.tensor([900, 333, 64], dtype=torch.int32, device="cuda")
        pool, table, _ = filled(fmt, lens.tolist())
        q = _queries(fmt, 3, gqa, nq)
        out = torch.zeros((3, 2, table.shape[1] * 16), device="cuda")
        kw = dict(scale=scale_of(fmt), out=out)
        ops.attention_mass(fmt, pool, q, table, lens, **kw)
        graph = torch.cuda.CUDAGraph()
        stream = torch.cuda.Stream()
        stream.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(stream), torch.cuda.graph(graph, stream=stream):
            ops.attention_mass(fmt, pool, q, table, lens, **kw)
        torch.cuda.current_stream().wait_stream(stream)
        for k in range(4):
            q.copy_(_queries(fmt, 3, gqa, nq, 50 + k))
            lens.copy_(torch.tensor([900 - 7 * k, 333 - 100 * k, 64 - 21 * k]))
            out.zero_()
            graph.replay()
            eager = ops.attention_mass(fmt, pool, q, table, lens, scale=scale_of(fmt))
            torch.cuda.synchronize()
            assert torch.equal(out, eager)


def test_a_query_that_is_not_finite_spoils_its_own_head_only():
    from pkv import ops

    for nq in (1, 8):
        fmt = _format(8, 128, 64)
        pool, table, _ = filled(fmt, [60, 60])
        q = _queries(fmt, 2, 4, nq)
        want = ops.attention_mass(fmt, pool, q, table, [60, 60], scale=0.1)
        q[0, 2, 0, 5] = float("nan")     # KV head 0 of sequence 0
        got = ops.attention_mass(fmt, pool, q, table, [60, 60], scale=0.1)
        assert torch.isnan(got[0, 0, :60 - nq + 1]).all()
        assert torch.equal(got[0, 1], want[0, 1]) and torch.equal(got[1], want[1])
        # ... and none at all where its row is not live
        dead = ops.attention_mass(fmt, pool, q, table, [60, 60], scale=0.1, widths=[0, nq])
        assert not dead[0].any() and torch.equal(dead[1], want[1])


def test_another_stream():
    from pkv import ops

    fmt = _format(8, 128, 64)
    pool, table, _ = filled(fmt, [500, 20])
    q = _queries(fmt, 2, 4, 1)
    lens = torch.tensor([500, 20], dtype=torch.int32, device="cuda")
    want = ops.attention_mass(fmt, pool, q, table, lens, scale=0.1)
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = []
    for s in streams:
        with torch.cuda.stream(s):
            got.append(ops.attention_mass(fmt, pool, q, table, lens, scale=0.1))
    torch.cuda.synchronize()
    assert all(torch.equal(g, want) for g in got)


def test_few_rows_under_a_table_too_wide_to_keep_scores():
    """The scores of 8 sequences under a table of 2^23 tokens each would take 4 GiB: K is
    read twice instead, with the same sums."""
    from pkv import ops

    fmt = _format(8, 128, 64, 128, 4)
    lens = [300, 17, 0, 1, 1000, 129, 256, 40]
    pool, table, _ = filled(fmt, lens)
    q = _queries(fmt, 8, 2, 1)
    wide = torch.full((8, 1 << 16), -1, dtype=torch.int32, device="cuda")
    wide[:, :table.shape[1]] = table
    out = [torch.zeros((8, 4, 1024), device="cuda") for _ in range(2)]
    want, bound = mass64(fmt, pool, table, lens, q, scale_of(fmt))
    for t, o in zip((table, wide), out):
        ops.attention_mass(fmt, pool, q, t, lens, scale=scale_of(fmt), out=o)
        got = o.double().cpu().numpy()
        for b, n in enumerate(lens):
            assert np.all(np.abs(got[b, :, :n] - want[b]) <= bound[b])


@pytest.mark.parametrize("nq", [1, 12])
def test_many_sequences(nq):
    """More sequences than a wave has lanes, many of them empty, behind and between the others."""
    fmt = _format(4, 64, 32, 16, 2)
    rng = np.random.default_rng(nq)
    lens = [int(n) if rng.random() < 0.6 else 0 for n in rng.integers(1, 700, 150)]
    lens[70:130] = [0] * 60
    lens[-3:] = [0] * 3
    _check(fmt, lens, 2, nq)


@pytest.mark.parametrize("scale", [-0.2, 0.0, 1e-30])
@pytest.mark.parametrize("nq,gqa", [(1, 2), (9, 2)])
def test_scales(scale, nq, gqa):
    from pkv import ops

    for bits in (8, 16):
        fmt = _format(bits, 64, 32)
        pool, table, _ = filled(fmt, [90, 33])
        q = _queries(fmt, 2, gqa, nq)
        want, bound = mass64(fmt, pool, table, [90, 33], q, scale)
        got = ops.attention_mass(fmt, pool, q, table, [90, 33], scale=scale).double().cpu().numpy()
        for b, n in enumerate((90, 33)):
            assert np.all(np.abs(got[b, :, :n] - want[b]) <= bound[b])
    with pytest.raises(ValueError):
        ops.attention_mass(fmt, pool, q, table, [90, 33], scale=float("nan"))


def test_python_refusals():
    from pkv import ops
    from pkv.cache_errors import CacheCapacityError
    from pkv.modes import ModelCapabilityUnsupported

    fmt = _format(8, 64, 32)
    pool, table, _ = filled(fmt, [40, 9])
    q = _queries(fmt, 2, 2, 1)
    out = torch.zeros((2, 2, 64), device="cuda")
    good = dict(scale=0.1, out=out)
    bad = [dict(out=out.double()), dict(out=out[:1]), dict(out=out[:, :1]), dict(out=out.transpose(1, 2)),
           dict(out=out, mass=torch.zeros((2, 2, 63), device="cuda")), dict(rows=[0]), dict(counted=[1, 2, 3]),
           dict(widths=[1]), dict(q_pos=[1]), dict(out=out.cpu()),
           dict(workspace=torch.zeros(1 << 20, device="cuda"))]
    for kw in bad:
        with pytest.raises(ValueError):
            ops.attention_mass(fmt, pool, q, table, [40, 9], **{**good, **kw})
    with pytest.raises(ValueError):
        ops.attention_mass(fmt, pool[:, :100].contiguous(), q, table, [40, 9], **good)
    with pytest.raises(ValueError):
        ops.attention_mass(fmt, pool, q.half(), table, [40, 9], **good)
    with pytest.raises(CacheCapacityError):
        ops.attention_mass(fmt, pool, q, table, [40, 9], workspace=torch.zeros(16, dtype=torch.uint8, device="cuda"),
                           **good)
    logits, scores = torch.zeros((1, 2, 100), device="cuda"), torch.zeros((1, 2), device="cuda")
    for kw in (dict(count=0), dict(count=201), dict(count=4, done=scores), dict(count=4, done=scores > 0, pad_token=100)):
        with pytest.raises((ValueError, ModelCapabilityUnsupported)):
            ops.beam_select(logits, scores, **kw)
    with pytest.raises(ModelCapabilityUnsupported):
        ops.beam_select(logits, scores, 65)
    with pytest.raises(ValueError):
        ops.beam_select(logits, scores[:, :1], 4)
    with pytest.raises(ValueError):
        ops.reorder_rows(torch.zeros((4, 6), device="cuda")[:, :3], [0], [1])
    with pytest.raises(ModelCapabilityUnsupported):
        ops.reorder_rows(torch.zeros((4, 6), device="cuda"), list(range(8193)), [1] * 8193)
    kept = torch.zeros((2, 2, 4), dtype=torch.int32, device="cuda")
    for kw in (dict(kept=kept[:, :1].contiguous()), dict(kept=kept.float()), dict(new_lens=[1]), dict(dst=table[:1])):
        a = dict(dict(kept=kept, new_lens=[4, 4], dst=table), **kw)
        with pytest.raises(ValueError):
            ops.evict_pages(fmt, pool, a["kept"], a["new_lens"], table, a["dst"])
