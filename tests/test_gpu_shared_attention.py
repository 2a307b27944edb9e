"""GPU: attention of sequences that share prefixes against the same in 64 bits, every
sequence by itself, over the pages' stored values."""

from __future__ import annotations

import numpy as np
import pytest

from step_case import paged64, side64

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")


@pytest.fixture(scope="module", autouse=True)
def _gpu():
    if not torch.cuda.is_available():
        pytest.skip("no GPU")


def _format(bits, dim, group=32, page=16, hk=2, dtype=torch.bfloat16):
    from pkv import ops

    return ops.PageFormat(hk, dim, page, bits, group, dtype)


def _cache(fmt, groups, *, seed=0, k_scale=1.0, spare=2):
    """Pages of ``groups = [(shared tokens, [own tokens, ...]), ...]``: whole shared pages are
    one page, a begun one is a copy in every sequence.  ``(pool, table, lens, members,
    group_starts, prefix_lens)`` with the sequences in shuffled order."""
    from pkv import ops

    rng = np.random.default_rng(seed)
    p = fmt.page_tokens
    total = sum(len(own) for _, own in groups)
    lens = [shared + n for shared, own in groups for n in own]
    width = max(max(-(-n // p) for n in lens), 1) + 1
    ids = rng.permutation(total * width + spare).astype(np.int32)
    place = rng.permutation(total)
    at = 0
    table = np.full((total, width), -1, np.int32)
    pool = ops.allocate_pool(fmt, len(ids))
    pool.fill_(0xFF)
    members, starts, row = [], [0], 0
    gen = torch.Generator().manual_seed(seed + 7)
    longest = max(max(lens), 1)
    sides = torch.randn((2, total, fmt.num_kv_heads, longest, fmt.head_dim), generator=gen)
    sides[0] *= k_scale
    for shared, own in groups:
        first = ids[at:at + shared // p]
        at += len(first)
        for i, n in enumerate(own):
            b = int(place[row])
            count = -(-(shared + n) // p)
            table[b, :len(first)] = first
            table[b, len(first):count] = ids[at:at + count - len(first)]
            at += count - len(first)
            if i:
                sides[:, b, :, :shared] = sides[:, members[-i], :, :shared]
            members.append(b)
            row += 1
        starts.append(row)
    by_place = np.zeros(total, np.int32)
    by_place[place] = lens
    sides = sides.to(fmt.dtype).cuda()
    table, lens = torch.from_numpy(table).cuda(), torch.from_numpy(by_place).cuda()
    ops.append_quantize(fmt, pool, sides[0].contiguous(), sides[1].contiguous(), table, torch.zeros_like(lens), lens)
    return pool, table, lens, members, starts, [shared for shared, _ in groups]


def _queries(fmt, batch, gqa, nq, seed=1, gain=1.0):
    gen = torch.Generator().manual_seed(seed)
    q = torch.randn((batch, fmt.num_kv_heads * gqa, nq, fmt.head_dim), generator=gen) * gain
    return q.cuda().to(fmt.dtype)


def _check(fmt, groups, gqa, nq, *, seed=0, gain=1.0, k_scale=1.0, q_pos=None, widths=None, unmap=(), prefix=None):
    from pkv import ops

    pool, table, lens, members, starts, prefixes = _cache(fmt, groups, seed=seed, k_scale=k_scale)
    for b, page in unmap:
        table[b, page] = -1
    batch = table.shape[0]
    q = _queries(fmt, batch, gqa, nq, seed + 1, gain)
    scale = fmt.head_dim ** -0.5
    want, bound = paged64(fmt, pool, table, lens, q, scale, q_pos=q_pos, widths=widths)
    got = ops.shared_prefix_attention(fmt, pool, q, table, lens, members, starts, prefixes if prefix is None else prefix,
                                      scale=scale, q_pos=q_pos, widths=widths)
    off = np.abs(got.double().cpu().numpy() - want)
    assert np.all(off <= bound), (float((off / bound).max()), np.argwhere(~(off <= bound))[0].tolist())
    return pool, table, lens, q, got


GROUPS = [(64, [1, 5, 30]), (0, [20]), (130, [3, 70, 17, 1, 100]), (33, [12])]


@pytest.mark.parametrize("dtype", ["bfloat16", "float16"])
@pytest.mark.parametrize("bits,dim,group", [
    (8, 64, 32), (8, 64, 64), (8, 128, 32), (8, 128, 64), (8, 128, 128), (8, 256, 32), (8, 256, 64), (8, 256, 128),
    (4, 64, 32), (4, 64, 64), (4, 128, 32), (4, 128, 64), (4, 128, 128), (4, 256, 32), (4, 256, 64), (4, 256, 128),
    (16, 64, 32), (16, 128, 32), (16, 256, 32), (8, 80, 32), (4, 37, 32), (16, 100, 32), (16, 7, 32), (8, 1, 32)])
@pytest.mark.parametrize("gqa,nq", [(4, 1), (8, 1), (1, 1), (2, 5), (3, 4)])
def test_layouts(bits, dim, group, dtype, gqa, nq):
    _check(_format(bits, dim, group, 16, 2, getattr(torch, dtype)), GROUPS, gqa, nq)


@pytest.mark.parametrize("page", [16, 32, 64, 128])
@pytest.mark.parametrize("bits", [4, 8, 16])
@pytest.mark.parametrize("gqa,nq", [(4, 1), (8, 4)])
def test_pages_and_lengths(page, bits, gqa, nq):
    for shared in (0, 1, 15, 16, 17, 31, 32, 127, 128, 500, 1025):
        _check(_format(bits, 128, 64, page, 1), [(shared, [1, 2, 16, 33, 129]), (shared + 1, [1, 300])], gqa, nq)


@pytest.mark.parametrize("bits", [4, 8, 16])
@pytest.mark.parametrize("members", [1, 2, 3, 8, 9, 17, 40])
@pytest.mark.parametrize("gqa,nq", [(4, 1), (7, 1), (16, 2)])
def test_members(bits, members, gqa, nq):
    """Rows of a group that fill one block, begin another, or leave a block short."""
    own = [1 + (11 * i) % 50 for i in range(members)]
    _check(_format(bits, 64, 64, 16, 2), [(150, own), (90, own[:2])], gqa, nq)


@pytest.mark.parametrize("bits", [4, 8, 16])
@pytest.mark.parametrize("gqa,nq", [(8, 1), (2, 3), (4, 8)])
def test_rows_that_see_little(bits, gqa, nq):
    """Positions of any order, before the first token (nothing is seen), inside the shared
    tokens, past the last; widths from none to all; pages that are not mapped."""
    fmt = _format(bits, 128, 64)
    groups = [(70, [5, 70, 300]), (100, [1, 40])]
    rng = np.random.default_rng(nq)
    q_pos = rng.integers(-3, 420, (5, nq)).astype(np.int32)
    q_pos[3], q_pos[4, 0] = -1, 20
    at = torch.from_numpy(q_pos).cuda()
    _check(fmt, groups, gqa, nq, q_pos=at)
    _check(fmt, groups, gqa, nq, widths=[nq, 0, max(1, nq // 2), 1, nq])
    _check(fmt, groups, gqa, nq, q_pos=at, widths=[nq, 1, nq - 1, nq, 0])
    # the same page missing in every sequence of a group; one sequence's own page
    _check(fmt, [(70, [5, 70, 300])], gqa, nq, unmap=[(0, 2), (1, 2), (2, 2)])
    _check(fmt, [(70, [40, 70, 300])], gqa, nq, unmap=[(1, 5), (0, 4), (2, 6)], q_pos=torch.from_numpy(q_pos[:3]).cuda())


@pytest.mark.parametrize("bits", [4, 8, 16])
@pytest.mark.parametrize("gain,k_scale", [(30.0, 1.0), (1e4, 1e-4), (1e-6, 1.0), (3.0, 8.0)])
def test_sharp_and_flat_weights(bits, gain, k_scale):
    _check(_format(bits, 128, 64), [(200, [40, 300, 7])], 4, 1, gain=gain, k_scale=k_scale)
    _check(_format(bits, 128, 64, dtype=torch.float16), [(200, [40, 300, 7])], 4, 2, gain=min(gain, 100.0), k_scale=k_scale)


@pytest.mark.parametrize("bits", [4, 16])
@pytest.mark.parametrize("groups", [
    [(100, [1 + 7 * i % 40 for i in range(64)])], [(100, [1 + 7 * i % 40 for i in range(65)])],
    [(40, [3, 20])] * 31 + [(0, [9])], [(40, [3, 20])] * 31 + [(0, [9]), (0, [2])], [(0, [5])] * 63, [(0, [5])] * 64,
    [(48, [2, 30, 17])] * 33, [(16, [1 + i % 3, 20]) for i in range(70)], [(3000, [10] * 8)] * 12],
    ids=lambda g: f"{len(g)}-{sum(len(own) for _, own in g)}")
def test_many_members_and_groups(bits, groups):
    """Up to 64 members in 63 groups each wave lays the call out by itself, beyond by a plan."""
    _check(_format(bits, 64, 32, 16, 1), groups, 4, 1)


def test_long_prefixes():
    """Runs of many pairs, more than a wave's page window."""
    _check(_format(8, 64, 64, 16, 1), [(20000, [100, 3000, 1])], 2, 1)
    _check(_format(4, 128, 64, 32, 1), [(17000, [10] * 12), (9000, [1, 2])], 4, 1)
    _check(_format(16, 64, 32, 128, 1), [(0, [9000, 20])], 4, 2)


def test_less_may_be_shared_than_is():
    """Any number of tokens up to what the sequences hold alike, and more than they hold."""
    fmt = _format(8, 128, 64)
    whole = [(64, [5, 20, 33])]
    for n in (0, 1, 16, 47, 63, 64):
        _check(fmt, whole, 4, 1, prefix=[n])
    _check(fmt, [(64, [0, 0, 0])], 4, 1, prefix=[500])
    _check(fmt, whole, 4, 1, prefix=[-5])


def test_against_paged_attention():
    """The framework's own attention over the same call, within the sum of both errors."""
    from pkv import ops

    for bits in (4, 8, 16):
        fmt = _format(bits, 128, 64, 16, 4)
        pool, table, lens, members, starts, prefix = _cache(fmt, [(300, [10, 20, 400, 5]), (64, [1, 2])])
        q = _queries(fmt, 6, 4, 1)
        scale = 128 ** -0.5
        one = ops.paged_attention(fmt, pool, q, table, lens, scale=scale)
        two = ops.shared_prefix_attention(fmt, pool, q, table, lens, members, starts, prefix, scale=scale)
        _, bound = paged64(fmt, pool, table, lens, q, scale)
        off = (one.double() - two.double()).abs().cpu().numpy()
        assert np.all(off <= 2 * bound)


def test_sequences_of_no_group():
    from pkv import ops

    fmt = _format(8, 64, 64)
    pool, table, lens, members, starts, prefix = _cache(fmt, [(50, [10, 20, 30]), (20, [5, 6])])
    q = _queries(fmt, 5, 4, 1)
    scale = 0.125
    whole = ops.shared_prefix_attention(fmt, pool, q, table, lens, members, starts, prefix, scale=scale)
    out = torch.full_like(q, 9.0)
    got = ops.shared_prefix_attention(fmt, pool, q, table, lens, members[:3], starts[:2], prefix[:1], scale=scale, out=out)
    assert got is out
    rest = members[3:]
    assert bool((out[rest] == 9.0).all())
    assert torch.equal(out[members[:3]], whole[members[:3]])
    fresh = ops.shared_prefix_attention(fmt, pool, q, table, lens, members[3:], [0, 2], prefix[1:], scale=scale)
    assert bool((fresh[members[:3]] == 0).all()) and bool((fresh[rest] != 0).any())
    # ids out of range and starts that leave members out are skipped
    ids = torch.tensor(members[:3] + [77, -1], dtype=torch.int32, device="cuda")
    out.fill_(9.0)
    ops.shared_prefix_attention(fmt, pool, q, table, lens, ids, [0, 3, 5], [50, 20], scale=scale, out=out)
    assert bool((out[rest] == 9.0).all()) and torch.equal(out[members[:3]], whole[members[:3]])
    out.fill_(9.0)
    ops.shared_prefix_attention(fmt, pool, q, table, lens, members, [3, 5], prefix[1:], scale=scale, out=out)
    assert bool((out[members[:3]] == 9.0).all()) and not bool((out[rest] == 9.0).all())


@pytest.mark.parametrize("bits,dtype", [(8, "bfloat16"), (4, "float16"), (16, "bfloat16"), (16, "float16")])
def test_later_tokens_that_are_not_finite(bits, dtype):
    """What a row may not see yet, its own sequence's later drafts or another's tokens,
    changes nothing for it."""
    from pkv import ops

    fmt = _format(bits, 128, 64, dtype=getattr(torch, dtype))
    pool, table, lens, members, starts, prefix = _cache(fmt, [(64, [30, 40, 8])])
    nq = 4
    q = _queries(fmt, 3, 4, nq)
    scale = 0.1
    clean = ops.shared_prefix_attention(fmt, pool, q, table, lens, members, starts, prefix, scale=scale)
    for bad in (float("nan"), float("inf"), -float("inf")):
        dirty = pool.clone()
        b = members[1]
        n = int(lens[b])
        token = torch.randn((3, fmt.num_kv_heads, 1, 128), device="cuda").to(fmt.dtype)
        token[:, :, :, 3] = bad
        where = lens.clone() - 2  # the last but one token of sequence b
        ops.append_quantize(fmt, dirty, token, token, table, where, [int(i == b) for i in range(3)])
        got = ops.shared_prefix_attention(fmt, dirty, q, table, lens, members, starts, prefix, scale=scale)
        others = [i for i in range(3) if i != b]
        assert torch.equal(got[others], clean[others])
        assert torch.equal(got[b, :, :nq - 2], clean[b, :, :nq - 2])
        # (the quantizer stores a NaN as a number: what counts is what the page holds)
        held = side64(fmt, dirty, table[b, :-(-n // 16)].tolist(), True)[:, n - 2, 3]
        seen = torch.isfinite(got[b, :, nq - 2:, 3]).cpu().numpy().reshape(fmt.num_kv_heads, -1)
        assert np.all(seen == np.isfinite(held)[:, None])


@pytest.mark.parametrize("bits", [4, 8, 16])
@pytest.mark.parametrize("dtype", ["bfloat16", "float16"])
def test_queries_that_are_not_numbers(bits, dtype):
    """A query with a NaN has a NaN result, in its row alone."""
    from pkv import ops

    fmt = _format(bits, 128, 64, dtype=getattr(torch, dtype))
    pool, table, lens, members, starts, prefix = _cache(fmt, [(300, [30, 400, 8]), (0, [50])])
    q = _queries(fmt, 4, 4, 2)
    call = lambda: ops.shared_prefix_attention(fmt, pool, q, table, lens, members, starts, prefix, scale=0.1)
    want = call()
    rows = [(0, 0, 1), (1, 5, 0), (3, 7, 1), (2, 3, 0)]
    for at in rows:
        q[at][9] = float("nan")
    got = call()
    for at in rows:
        assert bool(got[at].isnan().all())
        got[at] = want[at]
    assert torch.equal(got, want)


def test_starts_that_fall():
    """Groups that would overlap name no sequence."""
    from pkv import ops

    fmt = _format(8, 64, 64)
    pool, table, lens, members, starts, prefix = _cache(fmt, [(50, [10, 20, 30])])
    q = _queries(fmt, 3, 4, 1)
    ids = torch.tensor(members, dtype=torch.int32, device="cuda")
    for at in ([0, 3, 1, 3], [2, 0, 3, 3], [0, 2, 3, -5]):
        out = torch.full_like(q, 9.0)
        ops.shared_prefix_attention(fmt, pool, q, table, lens, ids, at, [48, 48, 48], scale=0.1, out=out)
        assert bool((out == 9.0).all())


def test_others_of_a_whole_batch_are_zeros():
    """As many members as sequences, one of them out of range: the rows of the sequence that
    none names are zeros, whatever the memory of the result held."""
    from pkv import ops

    fmt = _format(8, 64, 64)
    pool, table, lens, members, starts, prefix = _cache(fmt, [(50, [10, 20, 30])])
    q = _queries(fmt, 3, 4, 1)
    for ids, at, left in ((members[:2] + [-1], [0, 3], members[2]), (members, [1, 3], members[0])):
        ids = torch.tensor(ids, dtype=torch.int32, device="cuda")
        torch.full_like(q, 9.0)  # (memory that the call's result may take)
        got = ops.shared_prefix_attention(fmt, pool, q, table, lens, ids, at, prefix, scale=0.1)
        assert bool((got[left] == 0).all()) and bool((got != 9.0).all())
    for count in (0, 3):
        got = ops.shared_prefix_attention(fmt, pool, q, table, lens, members[:count], [0], [], scale=0.1)
        assert bool((got == 0).all())


def test_repeats_and_workspaces():
    """The same bits each time, in a workspace that held anything."""
    from pkv import ops

    fmt = _format(8, 128, 64)
    pool, table, lens, members, starts, prefix = _cache(fmt, [(700, [10, 500, 30]), (64, [1, 2])])
    q = _queries(fmt, 5, 4, 1)
    first = ops.shared_prefix_attention(fmt, pool, q, table, lens, members, starts, prefix, scale=0.1)
    from pkv import _native as nat

    need = nat.load().pkv_shared_attention_workspace_bytes(fmt.c_layout, 8, 1, 5, 2)
    work = torch.full((need,), 0xFF, dtype=torch.uint8, device="cuda")
    for _ in range(3):
        again = ops.shared_prefix_attention(fmt, pool, q, table, lens, members, starts, prefix, scale=0.1, workspace=work)
        assert torch.equal(first, again)


def test_refusals():
    from pkv import ops
    from pkv.cache_errors import CacheCapacityError
    from pkv.modes import ModelCapabilityUnsupported

    fmt = _format(8, 64, 64)
    pool, table, lens, members, starts, prefix = _cache(fmt, [(50, [10, 20, 30])])
    q = _queries(fmt, 3, 4, 1)

    def call(fmt=fmt, pool=pool, q=q, table=table, lens=lens, members=members, starts=starts, prefix=prefix, scale=0.1, **kw):
        return ops.shared_prefix_attention(fmt, pool, q, table, lens, members, starts, prefix, scale=scale, **kw)

    call()
    for bad in (dict(q=q[0]), dict(q=q.half()), dict(q=q.cpu()), dict(table=table[:2]), dict(lens=lens[:2]),
                dict(members=[0, 1, 1]), dict(starts=[0]), dict(prefix=[1, 2]), dict(scale=float("inf")),
                dict(pool=pool[:, :100].contiguous()), dict(out=q.float()), dict(widths=[1]),
                dict(workspace=torch.zeros(10, device="cuda")), dict(q=q[:, :3].contiguous())):
        with pytest.raises(ValueError):
            call(**bad)
    with pytest.raises(CacheCapacityError):
        call(workspace=torch.zeros(16, dtype=torch.uint8, device="cuda"))
    with pytest.raises(ModelCapabilityUnsupported):
        call(q=_queries(fmt, 3, 4, 9))
