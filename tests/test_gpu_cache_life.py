"""GPU: the operators that decide which cached state lives on, together over a device
arena: steps that append, attend and add up attention weight, beam selection, reordering
of the slots, eviction.  A plain model on the host holds, per slot, layer and KV head, the
stored bytes and the weight of every token."""

from __future__ import annotations

import math
import random

import numpy as np
import pytest

from cache_ops_case import mass64, scale_of
from test_gpu_evict import _plain, _tokens

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")


@pytest.fixture(scope="module", autouse=True)
def _gpu():
    if not torch.cuda.is_available():
        pytest.skip("no GPU")


class Model:
    """What the slots must hold: tokens[layer][slot][head] rows of bytes, one per part."""

    def __init__(self, arena):
        self.arena = arena
        self.held = {}

    def read(self, layer, slot):
        n = self.arena.lengths[slot]
        ids = self.arena.pages(slot) or [0]
        return [x[:, :n] for x in _tokens(self.arena.fmt, self.arena.pools[layer], ids)]

    def take(self, slots):
        for layer in range(len(self.arena.pools)):
            for s in slots:
                self.held[layer, s] = self.read(layer, s)

    def check(self, slots):
        for layer in range(len(self.arena.pools)):
            for s in slots:
                for x, y in zip(self.read(layer, s), self.held[layer, s]):
                    assert np.array_equal(x, y), (layer, s)

    def evict(self, slots, keep, sinks, recent):
        """The kept lists, by the device's weights; call before the arena's."""
        mass = self.arena.mass.cpu().numpy()
        sums = {}
        for layer in range(len(self.arena.pools)):
            for s in slots:
                n = self.arena.lengths[s]
                lists = [_plain(mass[layer, s, h], n, keep, sinks, recent) for h in range(mass.shape[2])]
                if n > keep:
                    self.held[layer, s] = [np.stack([x[h, k] for h, k in enumerate(lists)])
                                           for x in self.held[layer, s]]
                    sums[layer, s] = np.stack([mass[layer, s, h][k] for h, k in enumerate(lists)])
                else:
                    sums[layer, s] = mass[layer, s, :, :n]
        return sums


def _arena(bits=8, capacity=300, slots=12, layers=2, hk=2, page=16, dtype=torch.bfloat16):
    from pkv import ops
    from pkv.device_arena import DevicePageArena

    fmt = ops.PageFormat(hk, 64, page, bits, 32, dtype)
    arena = DevicePageArena(fmt, capacity, num_layers=layers, max_slots=slots, max_tokens=256)
    arena.track_mass()
    return arena


def _step(arena, slots, width, gqa, gen):
    """One append + attend of every slot and layer; the queries per layer."""
    from pkv.device_arena import DeviceBatchCache

    fmt = arena.fmt
    res = arena.reserve(slots, [width] * len(slots))
    queries = []
    for layer in range(len(arena.pools)):
        def rows(heads):
            return torch.randn((len(slots), heads, width, fmt.head_dim), generator=gen).cuda().to(fmt.dtype)

        q = rows(fmt.num_kv_heads * gqa)
        DeviceBatchCache(arena, layer, res).attend(q, rows(fmt.num_kv_heads), rows(fmt.num_kv_heads),
                                                   scale=scale_of(fmt))
        queries.append(q)
    return res, queries


@pytest.mark.parametrize("bits", [4, 8, 16])
def test_beams_with_eviction(bits):
    from pkv import ops

    gen, rng = torch.Generator().manual_seed(bits), random.Random(bits)
    beams, groups, gqa, vocab = 4, 2, 4, 501
    arena = _arena(bits)
    model = Model(arena)
    slots = [arena.open_slot() for _ in range(beams * groups)]
    # a prompt per group, shared by its beams
    heads = slots[::beams]
    _step(arena, heads, 45, gqa, gen)
    for g in range(groups):
        arena.fork([heads[g]] * 1, [slots[g * beams + 1]])
        arena.fork([heads[g]], [slots[g * beams + 2]])
        arena.fork([heads[g]], [slots[g * beams + 3]])
    model.take(slots)
    mass = arena.mass.cpu().numpy()
    for s in slots:
        assert np.array_equal(mass[:, s], mass[:, heads[slots.index(s) // beams]])
    scores = torch.zeros((groups, beams), device="cuda")
    slot_ids = torch.tensor(slots, dtype=torch.int32, device="cuda")
    for step in range(20):
        before = arena.mass.double().cpu().numpy()
        lens = [arena.lengths[s] for s in slots]
        res, queries = _step(arena, slots, 1, gqa, gen)
        for layer, q in enumerate(queries):
            want, bound = mass64(arena.fmt, arena.pools[layer], res.table, res.lens.tolist(), q,
                                 scale_of(arena.fmt))
            got = arena.mass[layer].double().cpu().numpy()
            for b, s in enumerate(slots):
                n = lens[b] + 1
                old = before[layer, s, :, :n].copy()
                old[:, lens[b]:] = 0
                assert np.all(np.abs(got[s, :, :n] - old - want[b]) <= bound[b] + 2.0 ** -24 * (old + want[b]))
        old_bytes = {k: v for k, v in model.held.items()}
        model.take(slots)
        for layer in range(len(arena.pools)):
            for b, s in enumerate(slots):
                for x, y in zip(model.held[layer, s], old_bytes[layer, s]):
                    assert np.array_equal(x[:, :lens[b]], y)
        # the best (beam, token) pairs, and the beams' state after their parents
        logits = torch.randn((groups, beams, vocab), generator=gen).cuda()
        scores, parents, _ = ops.beam_select(logits, scores, beams)
        sources = slot_ids.view(groups, beams).gather(1, parents.long()).flatten()
        host = sources.tolist()
        sums = arena.mass[:, host].clone()
        if step % 2:
            arena.reorder(slots, host)
        else:
            arena.reorder(slot_ids, sources)
            arena.sync_lengths()
        model.held.update({(l, s): x for l in range(len(arena.pools))
                           for s, x in zip(slots, [model.held[l, h] for h in host])})
        assert torch.equal(arena.mass[:, slots], sums)
        model.check(slots)
        if step % 6 == 5:
            some = rng.sample(slots, 7)           # with four spare slots: in two rounds
            evicted = arena.evicted.tolist()
            cut = {s: max(0, arena.lengths[s] - 40) for s in some}
            want = model.evict(some, 40, 3, 8)
            arena.evict(some, 40, sinks=3, recent=8)
            model.check(slots)
            for s in some:
                n = arena.lengths[s]
                assert n <= 40 and arena.evicted.tolist()[s] == evicted[s] + cut[s]
                for layer in range(len(arena.pools)):
                    assert np.array_equal(arena.mass[layer, s, :, :n].cpu().numpy(), want[layer, s])
    # nothing is lost or held twice
    refs = np.zeros(arena.capacity, int)
    for s in slots:
        for page in arena.pages(s):
            refs[page] += 1
    assert np.array_equal(refs, arena.refcounts().numpy())
    arena.release(slots)
    assert arena.status() == (arena.capacity, 0)
    assert not arena.evicted[:-1].any()


def test_eviction_without_room_changes_nothing():
    from pkv.cache_errors import CacheCapacityError

    gen = torch.Generator().manual_seed(1)
    arena = _arena(capacity=22, slots=6)
    a, b = arena.open_slot(), arena.open_slot()
    _step(arena, [a, b], 160, 2, gen)           # 10 pages each, 2 left
    model = Model(arena)
    model.take([a, b])
    mass = arena.mass.clone()
    with pytest.raises(CacheCapacityError):
        arena.evict([a, b], 60)
    model.check([a, b])
    assert torch.equal(arena.mass, mass) and arena.lengths[a] == arena.lengths[b] == 160
    assert arena.status() == (2, 0) and not arena.evicted.any()
    model.evict([a], 30, 4, 8)
    arena.evict([a], 30, sinks=4, recent=8)     # two pages are enough for this
    model.check([a, b])
    assert arena.status() == (10, 0)
    arena.evict([a, b], [0, 200])               # nothing of one, all of the other
    assert arena.lengths[a] == 0 and arena.lengths[b] == 160 and arena.lens[a].item() == 0
    model.check([b])


def test_eviction_refusals():
    from pkv.cache_errors import CacheCapacityError

    arena = _arena(slots=3)
    a, b = arena.open_slot(), arena.open_slot()
    arena.reserve([a, b], [40, 40])
    for bad in (dict(keep=-1), dict(keep=[1]), dict(keep=5, spare=[a]), dict(keep=5, spare=[])):
        with pytest.raises(ValueError):
            arena.evict([a, b], **bad)
    with pytest.raises(ValueError):
        arena.evict([a], torch.tensor([3]))
    full = arena.open_slot()
    with pytest.raises(CacheCapacityError):
        arena.evict([a, b], 10)                 # no spare slot
    arena.release([full])
    arena.evict([], 5)
    arena.evict([b], 10)
    assert arena.lengths[a] == 40 and arena.lengths[b] == 10
    plain = _arena()
    plain.mass = None
    with pytest.raises(ValueError):
        plain.evict([0], 5)


def test_a_runners_steps_with_eviction():
    """``DeviceRunner`` steps over a tracked arena: the same outputs as an untracked one
    while nothing is evicted; afterwards the positions go on, and a captured step gives
    what eager steps give."""
    from pkv import ops
    from pkv.device_arena import DevicePageArena, DeviceRunner
    from pkv.layer import AttentionStack, ModelSpec

    spec = ModelSpec(hidden=128, query_heads=4, kv_heads=2, head_dim=64, num_layers=2)
    model = AttentionStack(spec)
    fmt = ops.PageFormat(2, 64, 16, 8, 32, torch.bfloat16)
    gen = torch.Generator().manual_seed(3)
    prompt = torch.randn((2, 90, 128), generator=gen).cuda().to(torch.bfloat16)
    tokens = torch.randn((12, 2, 1, 128), generator=gen).cuda().to(torch.bfloat16)
    arenas = [DevicePageArena(fmt, 100, num_layers=2, max_slots=6, max_tokens=256) for _ in range(3)]
    outs = []
    for k, arena in enumerate(arenas):
        if k:
            arena.track_mass()
        runner = DeviceRunner(model, arena)
        slots = [arena.open_slot(), arena.open_slot()]
        got = [runner.execute(slots, prompt, [90, 50])]
        for i in range(4):
            got.append(runner.execute(slots, tokens[i]))
        if k:
            arena.evict(slots, 40, sinks=4, recent=16)
            assert arena.lengths[slots[0]] == arena.lengths[slots[1]] == 40
            assert arena.evicted[slots].tolist() == [54, 14]
            if k == 1:
                for i in range(4, 12):
                    got.append(runner.execute(slots, tokens[i]))
            else:
                got.append(runner.execute(slots, tokens[4]))
                hidden = tokens[5].clone()
                step = runner.capture_decode(slots, hidden, warm=False)
                for i in range(5, 12):
                    hidden.copy_(tokens[i])
                    step.replay()
                    got.append(step.out.clone())
                arena.sync_lengths()
            assert arena.lengths[slots[0]] == 48
            res = arena.reserve(slots, [0, 0])
            assert arena.positions(res).tolist() == [40 + 8 + 54, 40 + 8 + 14]
        outs.append(got)
    for x, y, z in zip(outs[0], outs[1], outs[2]):
        assert torch.equal(x, y) and torch.equal(x, z)
    for y, z in zip(outs[1][5:], outs[2][5:]):
        assert torch.allclose(y.float(), z.float(), atol=0.02, rtol=0.02)
    assert torch.allclose(arenas[1].mass[:, :, :, :48], arenas[2].mass[:, :, :, :48], atol=1e-2)


def test_attention_over_what_is_kept():
    """Outputs after an eviction against softmax attention in 64 bits over the kept
    tokens' stored values, each KV head with its own."""
    from pkv import ops
    from pkv.device_arena import DeviceBatchCache

    gen = torch.Generator().manual_seed(5)
    arena = _arena(bits=8, layers=1)
    slot = arena.open_slot()
    _step(arena, [slot], 150, 2, gen)
    arena.evict([slot], 50, sinks=2, recent=10)
    res = arena.reserve([slot], [1])
    fmt = arena.fmt
    q, k, v = (torch.randn((1, h, 1, 64), generator=gen).cuda().to(fmt.dtype) for h in (4, 2, 2))
    out = DeviceBatchCache(arena, 0, res).attend(q, k, v, scale=0.125)
    parts = ops.gather_pages(fmt, arena.pools[0], torch.tensor(arena.pages(slot), dtype=torch.int32, device="cuda"))
    kd, vd = (ops.dequantize_rows(parts[i:i + 3], 8, 64, 32).double() for i in (0, 3))
    kd, vd = (x.transpose(0, 1).flatten(1, 2)[:, :51] for x in (kd, vd))
    s = torch.softmax((q[0, :, 0].double().view(2, 2, 64) * 0.125) @ kd.transpose(1, 2).contiguous(), -1)
    want = (s @ vd.contiguous()).view(4, 64)
    assert (out[0, :, 0].double() - want).abs().max() < 2e-2      # the attention's own bound against its oracle
    assert math.isfinite(float(out.float().sum()))


def test_captured_eviction():
    """Growth and eviction as one graph over device operands, replayed between eager
    steps of another arena that does the same: the same tables, sums and pages."""
    arenas = [_arena(capacity=200, slots=8), _arena(capacity=200, slots=8)]
    slots = torch.arange(4, dtype=torch.int32, device="cuda")
    spare = torch.arange(4, 8, dtype=torch.int32, device="cuda")
    keep = torch.tensor([40, 25, 60, 0], dtype=torch.int32, device="cuda")
    grow = torch.full_like(slots, 9)
    for a in arenas:
        gen = torch.Generator().manual_seed(4)
        _step(a, [0, 1, 2, 3], 70, 2, gen)
    plain, graphed = arenas
    res = graphed.reserve(slots, torch.zeros_like(grow))
    warm = _arena(capacity=200, slots=8)
    warm.reserve(slots, grow)
    warm.evict(slots, keep, sinks=2, recent=5, max_keep=64, spare=spare)
    torch.cuda.synchronize()
    graph, stream = torch.cuda.CUDAGraph(), torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream), torch.cuda.graph(graph, stream=stream):
        graphed.reserve(slots, grow, out=res)
        graphed.evict(slots, keep, sinks=2, recent=5, max_keep=64, spare=spare)
    torch.cuda.current_stream().wait_stream(stream)
    for k in range(4):
        graph.replay()
        plain.reserve(slots, grow)
        plain.evict(slots, keep, sinks=2, recent=5, max_keep=64, spare=spare)
        torch.cuda.synchronize()
        for x, y in ((plain.table, graphed.table), (plain.lens, graphed.lens), (plain.state, graphed.state),
                     (plain.evicted, graphed.evicted), (plain.pools[1], graphed.pools[1])):
            assert torch.equal(x, y)
        n = plain.lens[:4].tolist()
        assert n == [40, 25, 60, 0]
        for s in range(4):
            assert torch.equal(plain.mass[:, s, :, :n[s]], graphed.mass[:, s, :, :n[s]])
    assert graphed.status()[1] == 0


def test_an_evicted_prompt_is_not_published():
    from pkv.device_cache import DevicePrefixIndex

    class Fingerprint:
        digest = "text"

    arena = _arena(slots=6)
    index = DevicePrefixIndex(arena, capacity_pages=20, max_entries=2)
    a, b = arena.open_slot(), arena.open_slot()
    gen = torch.Generator().manual_seed(1)
    _step(arena, [a, b], 100, 2, gen)
    arena.evict([a], 40)
    assert not index.publish(a, Fingerprint, list(range(100)))
    assert index.publish(b, Fingerprint, list(range(100)))


def test_rows_named_twice_are_refused():
    from pkv import ops

    state = torch.zeros((4, 8), device="cuda")
    with pytest.raises(ValueError):
        ops.reorder_rows(state, [1, 1], [0, 2])
    ops.reorder_rows(state, [1, -1, -1], [0, 2, 3])          # rows that do not exist are none
    mass = torch.zeros((4, 1, 16), device="cuda")
    with pytest.raises(ValueError):
        ops.evict_select(mass, [16, 16], 4, rows=[2, 2], with_mass=True)
    kept, _ = ops.evict_select(mass, [16, 16], 4, rows=[2, 2])
    assert torch.equal(kept[0], kept[1])
    fmt = ops.PageFormat(1, 64, 16, 8, 32, torch.bfloat16)
    pool = torch.zeros((2, fmt.page_bytes), dtype=torch.uint8, device="cuda")
    q = torch.zeros((2, 1, 1, 64), dtype=torch.bfloat16, device="cuda")
    with pytest.raises(ValueError):
        ops.attention_mass(fmt, pool, q, [[0], [1]], [5, 5], scale=1.0, mass=mass, rows=[1, 1])
