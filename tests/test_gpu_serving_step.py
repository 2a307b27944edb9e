"""GPU: rotation with append, attention over packed prompts and attention over shared
prefixes one after the other, as a serving step runs them: by themselves on an arena's
reservations, through the device runner, and captured."""

from __future__ import annotations

import numpy as np
import pytest

from step_case import assert_turned, attention64, attention_bound, half_step, paged64, turned64

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")


@pytest.fixture(scope="module", autouse=True)
def _gpu():
    if not torch.cuda.is_available():
        pytest.skip("no GPU")


def _arena(bits, dim=64, dtype=torch.bfloat16, hk=2, page=16, **kw):
    from pkv import ops
    from pkv.device_arena import DevicePageArena

    fmt = ops.PageFormat(hk, dim, page, bits, 32, dtype)
    return DevicePageArena(fmt, 400, max_slots=16, max_tokens=2048, **kw)


def _fork(arena, sources, slots):
    for a, b in zip(sources, slots):
        arena.fork([a], [b])


def _projection(rows, heads, fmt, seed, lead=()):
    gen = torch.Generator().manual_seed(seed)
    x = torch.randn((*lead, rows, (heads + 2 * fmt.num_kv_heads) * fmt.head_dim), generator=gen)
    return x.cuda().to(fmt.dtype)


def _frequencies(half):
    return (10000.0 ** (-torch.arange(half, dtype=torch.float64) / half)).float().cuda()


def _check_prompts(fmt, q, k, v, out, starts, scale):
    q64, k64, v64 = (t.double().cpu().numpy() for t in (q, k, v))
    got = out.double().cpu().numpy()
    gqa = q.shape[1] // k.shape[1]
    operand = half_step(fmt.dtype)
    for a, b in zip(starts, starts[1:]):
        for h in range(q.shape[1]):
            want, weight, terms = attention64(q64[a:b, h], k64[a:b, h // gqa], v64[a:b, h // gqa],
                                              np.arange(1, b - a + 1), scale)
            bound = attention_bound(want, weight, terms, scale, fmt.dtype, dim=fmt.head_dim, tokens=b - a,
                                    operand=operand)
            assert np.all(np.abs(got[a:b, h] - want) <= bound)


def _check_shared(arena, res, q, out, scale, width):
    want, bound = paged64(arena.fmt, arena.pools[0], res.table, res.lens, q, scale, widths=[width] * q.shape[0])
    assert np.all(np.abs(out.double().cpu().numpy() - want) <= bound)


@pytest.mark.parametrize("bits", [4, 8, 16])
@pytest.mark.parametrize("dtype", ["bfloat16", "float16"])
def test_prompts_forks_and_steps(bits, dtype):
    """Two prompts packed; answers forked from them, some a step ahead; steps of one and of
    three tokens over what they share, each against 64 bits over the pages it left."""
    from pkv import ops

    heads, dtype = 8, getattr(torch, dtype)
    arena = _arena(bits, dtype=dtype)
    fmt, scale, inv = arena.fmt, 0.125, _frequencies(32)
    prompts = [arena.open_slot(), arena.open_slot()]
    lens = [150, 37]
    starts = [0, 150, 187]
    qkv = _projection(187, heads, fmt, 1)
    res = arena.reserve(prompts, lens)
    q, k, v = ops.rope_append(fmt, arena.pools[0], qkv, res.table, res.starts, inv, heads, row_starts=starts, with_kv=True)
    places = np.concatenate([np.arange(n) for n in lens]).astype(np.float64)
    x = qkv.double().cpu().numpy().reshape(187, -1, 64)
    turned, size = turned64(x, places[:, None] * inv.double().cpu().numpy(), 32)
    assert_turned(q, turned[:, :heads], size[:, :heads], dtype)
    assert_turned(k, turned[:, heads:heads + 2], size[:, heads:heads + 2], dtype)
    assert torch.equal(v.flatten(1), qkv[:, -128:])
    _check_prompts(fmt, q, k, v, ops.prompt_attention(q, k, v, starts, scale=scale), starts, scale)
    answers = [arena.open_slot() for _ in range(5)]
    _fork(arena, [prompts[0]] * 3 + [prompts[1]] * 2, answers)
    batch = [answers[3], answers[0], prompts[0], answers[4], answers[1], answers[2]]
    groups = arena.prefix_groups(batch)
    sizes = {tuple(sorted(batch.index(s) for s in g)): n for g, n in (
        (answers[3:], 32), ([prompts[0], *answers[:3]], 144))}
    members, begins, prefix = (t.tolist() for t in groups)
    assert {tuple(sorted(members[a:b])): n for a, b, n in zip(begins, begins[1:], prefix)} == sizes
    assert arena.prefix_groups(batch, least=100)[2].tolist().count(0) == 1
    for step, width in enumerate((1, 3, 1)):
        qkv = _projection(width, heads, fmt, 10 + step, (len(batch),))
        before = list(arena.lengths)
        res = arena.reserve(batch, [width] * len(batch))
        q = ops.rope_append(fmt, arena.pools[0], qkv, res.table, res.starts, inv, heads)
        x = qkv.double().cpu().numpy().reshape(len(batch), width, -1, 64)
        places = np.array([[before[s] + i for i in range(width)] for s in batch], np.float64)
        turned, size = turned64(x, places[..., None] * inv.double().cpu().numpy(), 32)
        assert_turned(q.transpose(1, 2), turned[:, :, :heads], size[:, :, :heads], dtype)
        out = ops.shared_prefix_attention(fmt, arena.pools[0], q, res.table, res.lens, *groups, scale=scale)
        _check_shared(arena, res, q, out, scale, width)
    arena.check()


def _model(layers, dtype="bfloat16"):
    from pkv.layer import AttentionStack, ModelSpec

    return AttentionStack(ModelSpec(hidden=256, query_heads=8, kv_heads=2, head_dim=64, num_layers=layers,
                                    rope_theta=10000.0, dtype=dtype, vocab_size=100), seed=3)


def _hidden(rows, seed, lead=()):
    gen = torch.Generator().manual_seed(seed)
    return torch.randn((*lead, rows, 256), generator=gen).cuda().bfloat16()


def _near(got, want, layers):
    """Two bfloat16 runs of the same layers.  A layer rounds its projection, its turned heads,
    its attention and its output, and each run stores K and V by itself: six half steps of
    2^-8 of a row's size at the most per layer and run (random weights keep sizes, and a
    row's errors add up squared, as its elements do)."""
    off = (got.double() - want.double()).norm(dim=-1)
    size = want.double().norm(dim=-1)
    assert bool((off <= 12 * layers * 2.0 ** -8 * size).all()), float((off / size).max())


@pytest.mark.parametrize("bits", [8, 16])
def test_runner(bits):
    """Packed prompts and steps over shared prefixes through the device runner, beside the
    runner's ordinary steps on another arena."""
    from pkv.device_arena import DeviceRunner

    model = _model(2)
    one, two = _arena(bits, num_layers=2), _arena(bits, num_layers=2)
    shared, plain = DeviceRunner(model, one), DeviceRunner(model, two)
    lens = [90, 33, 1]
    slots = [one.open_slot() for _ in lens]
    assert [two.open_slot() for _ in lens] == slots
    packed = _hidden(sum(lens), 5)
    padded = torch.zeros((3, 90, 256), dtype=packed.dtype, device="cuda")
    at = 0
    for b, n in enumerate(lens):
        padded[b, :n] = packed[at:at + n]
        at += n
    got, want = shared.prefill(slots, packed, lens), plain.execute(slots, padded, lens)
    if bits == 16:    # (the other path reads quantized pages back)
        _near(got, torch.cat([want[b, :n] for b, n in enumerate(lens)]), 2)
    assert one.lengths == two.lengths
    forks = [one.open_slot() for _ in range(4)]
    assert [two.open_slot() for _ in range(4)] == forks
    for arena in (one, two):
        if bits == 8:    # (so that both start from the same pages)
            for a, b in zip(one.pools, two.pools):
                b.copy_(a)
            two.table.copy_(one.table)
        _fork(arena, [slots[0]] * 3 + [slots[1]], forks)
    batch = slots + forks
    groups = one.prefix_groups(batch)
    for step in range(3):
        x = _hidden(1 + step % 2, 20 + step, (7,))
        _near(shared.execute(batch, x, shared=groups), plain.execute(batch, x), 2)
    assert one.lengths == two.lengths
    with pytest.raises(ValueError):
        shared.prefill(slots, packed, lens)
    with pytest.raises(ValueError):
        shared.execute(batch[:6], _hidden(1, 30, (6,)), shared=groups)
    with pytest.raises(ValueError):
        shared.capture_decode(batch[:6], _hidden(1, 30, (6,)), shared=groups)
    fresh = one.open_slot()
    with pytest.raises(ValueError):
        shared.prefill([fresh], packed, [5])
    one.track_mass()
    from pkv.modes import ModelCapabilityUnsupported

    with pytest.raises(ModelCapabilityUnsupported):
        shared.prefill([fresh], packed[:5], [5])
    shared.execute(batch, _hidden(1, 30, (7,)), shared=groups)    # (sums and shared prefixes together)
    assert one.lengths[fresh] == 0
    one.check()


def test_captured_steps():
    """Two captured decode steps over shared prefixes of two halves of a batch, replayed in
    turn with eager work of their kind between them, each replay against an eager step
    on a second arena that holds the same."""
    from pkv.device_arena import DeviceRunner

    model = _model(2)
    one, two = _arena(8, num_layers=2), _arena(8, num_layers=2)
    captured, eager = DeviceRunner(model, one), DeviceRunner(model, two)
    for runner in (captured, eager):
        arena = runner.arena
        slots = [arena.open_slot() for _ in range(6)]
        runner.prefill(slots[:2], _hidden(130, 5), [100, 30])
        _fork(arena, [slots[0]] * 2 + [slots[1]] * 2, slots[2:])
    halves = ([slots[0], slots[2], slots[4]], [slots[1], slots[3], slots[5]])
    groups = [one.prefix_groups(half) for half in halves]
    assert groups[0][2].tolist()[0] == 96
    buffers = [_hidden(1, 40 + i, (3,)) for i in range(2)]
    steps = [captured.capture_decode(half, buffer, shared=group) for half, buffer, group in zip(halves, buffers, groups)]
    wants = [eager.execute(half, buffer, shared=group) for half, buffer, group in zip(halves, buffers, groups)]
    for turn in range(5):
        for i in (turn % 2, 1 - turn % 2):
            buffers[i].copy_(_hidden(1, 100 + 10 * turn + i, (3,)))
            steps[i].replay()
            want = eager.execute(halves[i], buffers[i], shared=groups[i])
            torch.cuda.synchronize()
            assert torch.equal(steps[i].out, want)
    one.sync_lengths()
    assert one.lengths == two.lengths
    one.check()
    assert len(wants) == 2


def test_another_stream():
    """Calls on a side stream, the tensors made there and used after it has been waited for."""
    from pkv import ops

    arena = _arena(8)
    fmt, inv = arena.fmt, _frequencies(32)
    slots = [arena.open_slot() for _ in range(3)]
    res = arena.reserve(slots, [20, 300, 7])
    starts = torch.tensor([0, 20, 320, 327], dtype=torch.int32, device="cuda")
    qkv = _projection(327, 8, fmt, 9)

    def run():
        q, k, v = ops.rope_append(fmt, arena.pools[0], qkv, res.table, res.starts, inv, 8, row_starts=starts, with_kv=True)
        out = ops.prompt_attention(q, k, v, starts, scale=0.125)
        last = torch.stack([q[n - 1] for n in (20, 320, 327)])[:, :, None].contiguous()
        return out, ops.shared_prefix_attention(fmt, arena.pools[0], last, res.table, res.lens, [0, 1, 2], [0, 3], [0],
                                                scale=0.125)

    want = run()
    torch.cuda.synchronize()
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        got = run()
    torch.cuda.current_stream().wait_stream(stream)
    assert all(torch.equal(a, b) for a, b in zip(got, want))


@pytest.mark.parametrize("bits", [4, 8, 16])
def test_pages_past_32_bits(bits):
    """Pages that lie beyond 4 GiB in their pool hold and give what pages of a small pool do."""
    from pkv import ops

    fmt = ops.PageFormat(8, 128, 128, bits, 64, torch.bfloat16)
    count = (9 << 29) // fmt.page_bytes + 8
    far, near = torch.empty((count, fmt.page_bytes), dtype=torch.uint8, device="cuda"), ops.allocate_pool(fmt, 8)
    far[-8:] = 0
    lens = torch.tensor([200, 330, 140], dtype=torch.int32, device="cuda")
    table = torch.tensor([[0, 1, -1], [0, 2, 3], [0, 4, -1]], dtype=torch.int32, device="cuda")
    zero, inv = torch.zeros_like(lens), _frequencies(64)
    qkv = _projection(670, 16, fmt, 1)
    qkv[200:328] = qkv[:128]    # the first page is one for all three
    qkv[530:658] = qkv[:128]
    last = _projection(1, 16, fmt, 2, (3,))
    got = []
    for pool, at in ((near, table), (far, torch.where(table < 0, table, table + count - 8))):
        q = ops.rope_append(fmt, pool, qkv, at, zero, inv, 16, row_starts=[0, 200, 530, 670])
        step = ops.rope_append(fmt, pool, last, at, lens, inv, 16)
        out = ops.shared_prefix_attention(fmt, pool, step, at, lens + 1, [0, 1, 2], [0, 3], [128], scale=0.1)
        got.append((q, step, out, pool[-8:][:5].clone()))
    for a, b in zip(*got):
        assert torch.equal(a, b)
    assert bool((got[0][2] != 0).any(-1).all())


def test_rows_past_32_bits():
    """Packed rows whose elements are numbered past 2^31: the last prompts as by themselves."""
    from pkv import ops

    rows, heads, dim = 540_000, 32, 128
    gen = torch.Generator(device="cuda").manual_seed(1)
    q = torch.empty((rows, heads, dim), dtype=torch.bfloat16, device="cuda")
    q[-9:] = torch.randn((9, heads, dim), generator=gen, device="cuda")
    q[:-9] = q[-1]
    k, v = (torch.randn((rows, 2, dim), generator=gen, device="cuda").bfloat16() for _ in range(2))
    starts = list(range(0, rows - 9, 30)) + [rows - 9, rows - 4, rows]
    out = ops.prompt_attention(q, k, v, starts, scale=0.1)
    want = ops.prompt_attention(*(t[-9:].contiguous() for t in (q, k, v)), [0, 5, 9], scale=0.1)
    assert torch.equal(out[-9:], want)
    some = slice(30 * 9000, 30 * 9001)
    assert torch.equal(out[some], ops.prompt_attention(*(t[some].contiguous() for t in (q, k, v)), [0, 30], scale=0.1))


def test_captured_prompts():
    """Rotation with append and prompt attention in a graph, replayed for other rows and other
    lengths with eager calls between, each replay against the eager calls."""
    from pkv import ops

    arena = _arena(8)
    fmt, inv, scale = arena.fmt, _frequencies(32), 0.125
    slots = [arena.open_slot() for _ in range(3)]
    res = arena.reserve(slots, [300, 300, 300])
    cuts = [[0, 100, 130, 300], [0, 1, 2, 300], [0, 0, 290, 300], [0, 64, 128, 256]]
    starts = torch.tensor(cuts[0], dtype=torch.int32, device="cuda")
    qkv = _projection(300, 8, fmt, 1)

    def run(pool):
        q, k, v = ops.rope_append(fmt, pool, qkv, res.table, res.starts, inv, 8, row_starts=starts, with_kv=True, out=held[0])
        return ops.prompt_attention(q, k, v, starts, scale=scale, out=held[1])

    shapes = [(300, 8, 64), (300, 2, 64), (300, 2, 64)]
    held = ([torch.zeros(s, dtype=fmt.dtype, device="cuda") for s in shapes], torch.zeros(shapes[0], dtype=fmt.dtype, device="cuda"))
    mine, pool = held, arena.pools[0]
    run(pool)
    torch.cuda.synchronize()
    graph, stream = torch.cuda.CUDAGraph(), torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        with torch.cuda.graph(graph, stream=stream):
            run(pool)
    torch.cuda.current_stream().wait_stream(stream)
    for turn in range(8):
        starts.copy_(torch.tensor(cuts[turn % 4], dtype=torch.int32))
        qkv.copy_(_projection(300, 8, fmt, 50 + turn))
        held = ([t.clone() for t in mine[0]], mine[1].clone())
        other = pool.clone()
        want = run(other)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(mine[1], want) and torch.equal(pool, other)
        assert all(torch.equal(a, b) for a, b in zip(mine[0], held[0]))


def test_steps_that_run_out_of_pages():
    """A prefill or a shared step without pages raises and changes neither lengths nor the
    tokens that the pages hold."""
    from pkv import ops
    from pkv.cache_errors import CacheCapacityError
    from pkv.device_arena import DevicePageArena, DeviceRunner
    from pkv.modes import ModelCapabilityUnsupported

    fmt = ops.PageFormat(2, 64, 16, 8, 32, torch.bfloat16)
    arena = DevicePageArena(fmt, 7, num_layers=2, max_slots=8, max_tokens=512)
    runner = DeviceRunner(_model(2), arena)
    a, b, c = (arena.open_slot() for _ in range(3))
    runner.prefill([a], _hidden(96, 1), [96])
    arena.fork([a], [b])
    held = [p[arena.pages(a)].clone() for p in arena.pools]
    with pytest.raises(CacheCapacityError):
        runner.prefill([c], _hidden(100, 2), [100])
    groups = arena.prefix_groups([a, b])
    assert groups[2].tolist() == [96]
    with pytest.raises(CacheCapacityError):
        runner.execute([a, b], _hidden(8, 3, (2,)), shared=groups)
    with pytest.raises(ModelCapabilityUnsupported):    # (more query rows than a shared step takes)
        runner.execute([a, b], _hidden(9, 3, (2,)), shared=groups)
    assert arena.lengths[:3] == [96, 96, 0] and arena.lens.tolist()[:3] == [96, 96, 0]
    assert all(torch.equal(p[arena.pages(a)], h) for p, h in zip(arena.pools, held))
    out = runner.execute([a], _hidden(2, 4, (1,)), shared=arena.prefix_groups([a]))
    assert bool(torch.isfinite(out).all()) and arena.lengths[:2] == [98, 96]
    arena.check()
