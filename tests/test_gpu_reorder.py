"""GPU: rows of state tensors and slots of the page arena that become others' copies,
all at once, against the same on the host."""

from __future__ import annotations

import random

import numpy as np
import pytest

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")


@pytest.fixture(scope="module", autouse=True)
def _gpu():
    if not torch.cuda.is_available():
        pytest.skip("no GPU")


def _state(shape, dtype, seed=0):
    gen = torch.Generator().manual_seed(seed)
    n = int(np.prod(shape)) * torch.empty(0, dtype=dtype).element_size()
    raw = torch.randint(0, 256, (n,), generator=gen, dtype=torch.uint8)
    return raw.view(dtype).view(shape).cuda()


def _check(shape, dtype, targets, sources, dim=0):
    from pkv import ops

    x = _state(shape, dtype)
    before = x.cpu().view(torch.uint8)
    rows = x.shape[dim]
    want = before.clone().view(*shape[:dim + 1], -1)
    old = want.clone()
    for t, s in zip(targets, sources):
        if 0 <= t < rows and 0 <= s < rows:
            want.select(dim, t).copy_(old.select(dim, s))
    assert ops.reorder_rows(x, targets, sources, dim=dim) is x
    assert torch.equal(x.cpu().view(torch.uint8).view(want.shape), want)


@pytest.mark.parametrize("dtype", [torch.uint8, torch.bfloat16, torch.float32, torch.int64])
@pytest.mark.parametrize("size", [1, 2, 3, 15, 16, 17, 1000, 1001, 4096, 33333])
def test_rows(dtype, size):
    rng = random.Random(size)
    n = 13
    perm = list(range(n))
    rng.shuffle(perm)
    _check((n, size), dtype, list(range(n)), perm)                             # a permutation
    _check((n, size), dtype, list(range(n)), [rng.randrange(n) for _ in range(n)])
    _check((n, size), dtype, perm[:5], [rng.randrange(n) for _ in range(5)])
    _check((3, n, size), dtype, perm[:6], [rng.randrange(n) for _ in range(6)], dim=1)
    _check((2, 3, n, size), dtype, perm, [rng.randrange(n) for _ in range(n)], dim=2)
    _check((n, size), dtype, [4], [9])
    _check((n, size), dtype, [], [])
    _check((n, size), dtype, [0, 1, 2, 50, 3], [1, 0, -1, 2, 13])              # rows that do not exist


@pytest.mark.parametrize("count,size", [(1, 100000), (256, 1000), (300, 4099), (512, 2064), (513, 33), (1000, 77), (4097, 40), (8192, 5)])
def test_many_rows(count, size):
    rng = random.Random(count)
    perm = list(range(count))
    rng.shuffle(perm)
    _check((count, size), torch.int16, perm, [rng.randrange(count) for _ in range(count)])


def test_rows_past_4_gib():
    from pkv import ops

    x = torch.zeros((5, (1 << 30) + 7), dtype=torch.uint8, device="cuda")
    for i in range(5):
        x[i] = i
    ops.reorder_rows(x, [0, 4, 2], [4, 0, 3])
    assert [int(x[i, -1]) for i in range(5)] == [4, 1, 3, 3, 0]
    assert [int(x[i, 0]) for i in range(5)] == [4, 1, 3, 3, 0]
    assert [int(x[i].max()) for i in range(5)] == [4, 1, 3, 3, 0]
    assert [int(x[i].min()) for i in range(5)] == [4, 1, 3, 3, 0]


# ---- arena slots ---------------------------------------------------------------------------


def _arena(capacity=64, slots=8, tokens=512, **kw):
    from pkv import ops
    from pkv.device_arena import DevicePageArena

    fmt = ops.PageFormat(1, 64, 16, 8, 32, torch.bfloat16)
    return DevicePageArena(fmt, capacity, max_slots=slots, max_tokens=tokens, **kw)


def _consistent(arena):
    """Reference counts, free pages and lengths agree with the tables."""
    table, lens = arena.table.cpu().numpy(), arena.lens.cpu().numpy()
    refs = np.zeros(arena.capacity, int)
    for s in range(arena.max_slots):
        n = -(-int(lens[s]) // arena.page_tokens)
        assert (table[s, :n] >= 0).all() and (table[s, n:] == -1).all(), s
        for page in table[s, :n]:
            refs[page] += 1
    assert np.array_equal(refs, arena.refcounts().numpy())
    assert sorted(arena.free_stack().tolist()) == [i for i in range(arena.capacity) if refs[i] == 0]
    assert lens.tolist() == arena.lengths
    assert arena.status()[1] == 0


def test_arena_reorder_by_steps():
    """Random growth, forks, cuts and reorderings; each reordering moves tables and
    lengths at once and frees what is left without an owner."""
    rng = random.Random(4)
    for capacity, slots, tokens in ((200, 8, 512), (3000, 70, 1100)):
        arena = _arena(capacity, slots, tokens)
        for step in range(40):
            kind = rng.random()
            if kind < 0.4:
                some = rng.sample(range(slots), rng.randint(1, slots))
                arena.reserve(some, [min(rng.randint(0, 40), tokens - arena.lengths[s]) for s in some])
                if arena.status()[1]:
                    arena.state[1:2].zero_()
                    arena.sync_lengths()
            elif kind < 0.5:
                some = rng.sample(range(slots), 2)
                arena.truncate(some, [rng.randint(0, arena.lengths[s]) for s in some])
            else:
                some = rng.sample(range(slots), rng.randint(1, slots))
                sources = [rng.randrange(slots) for _ in some]
                table, lens = arena.table.cpu(), arena.lens.cpu()
                arena.reorder(some, sources)
                table[some], lens[some] = table[sources], lens[sources]
                assert torch.equal(arena.table.cpu(), table) and torch.equal(arena.lens.cpu(), lens)
            _consistent(arena)


def test_arena_reorder_of_many_slots():
    rng = random.Random(3)
    arena = _arena(9000, 4096, 64)
    arena.reserve(list(range(4096)), [rng.randint(0, 33) for _ in range(4096)])
    table, lens = arena.table.cpu(), arena.lens.cpu()
    some = rng.sample(range(4096), 4096)
    sources = [rng.randrange(4096) for _ in some]
    arena.reorder(some, sources)
    table[some], lens[some] = table[sources], lens[sources]
    assert torch.equal(arena.table.cpu(), table) and torch.equal(arena.lens.cpu(), lens)
    _consistent(arena)
    arena.reorder([], [])


def test_arena_reorder_is_deterministic():
    """Two arenas through the same calls hand out the same pages."""
    stacks = []
    for _ in range(2):
        arena = _arena(4000, 64, 1024)
        rng = random.Random(1)
        arena.reserve(list(range(64)), [700 + s for s in range(64)])
        for _ in range(5):
            arena.reorder(list(range(64)), [rng.randrange(64) for _ in range(64)])
        stacks.append((arena.free_stack(), arena.table.cpu()))
        _consistent(arena)
    assert torch.equal(stacks[0][0], stacks[1][0]) and torch.equal(stacks[0][1], stacks[1][1])


def test_arena_reorder_of_slots_out_of_range():
    from pkv.cache_errors import CacheCorruptionError

    arena = _arena()
    arena.reserve([0, 1], [20, 40])
    slots = torch.tensor([0, 9, 2], dtype=torch.int32)
    arena.reorder(slots, torch.tensor([1, 0, -1], dtype=torch.int32))
    assert arena.lens.tolist()[:3] == [40, 40, 0]
    with pytest.raises(CacheCorruptionError):
        arena.check()
    arena.sync_lengths()
    _consistent(arena)


def test_arena_reorder_replays():
    """Growth and reordering captured together, replayed with other parents."""
    plain, graphed = _arena(400, 8), _arena(400, 8)
    slots = torch.arange(8, dtype=torch.int32, device="cuda")
    ones = torch.full_like(slots, 5)
    parents = torch.zeros_like(slots)
    for a in (plain, graphed):
        a.reserve(list(range(8)), [30 + 3 * s for s in range(8)])
    res = graphed.reserve(slots, torch.zeros_like(ones))
    graph, stream = torch.cuda.CUDAGraph(), torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream), torch.cuda.graph(graph, stream=stream):
        graphed.reserve(slots, ones, out=res)
        graphed.reorder(slots, parents)
    torch.cuda.current_stream().wait_stream(stream)
    rng = random.Random(2)
    for _ in range(6):
        choice = [rng.randrange(8) for _ in range(8)]
        parents.copy_(torch.tensor(choice, dtype=torch.int32))
        graph.replay()
        plain.reserve(list(range(8)), [5] * 8)
        plain.reorder(list(range(8)), choice)
        torch.cuda.synchronize()
        assert torch.equal(plain.table, graphed.table) and torch.equal(plain.lens, graphed.lens)
        assert torch.equal(plain.state, graphed.state)
    graphed.sync_lengths()
    _consistent(graphed)
