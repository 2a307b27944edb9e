"""GPU: a step over an emptied slot that is rolled back: the slot's text goes on where it
was, with the tokens evicted before it counted."""

from __future__ import annotations

import pytest

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")


@pytest.fixture(scope="module", autouse=True)
def _gpu():
    if not torch.cuda.is_available():
        pytest.skip("no GPU")


def test_positions_go_on_after_a_failed_step():
    from pkv import ops
    from pkv.device_arena import DevicePageArena, DeviceRunner
    from pkv.layer import AttentionStack, ModelSpec

    spec = ModelSpec(hidden=128, query_heads=4, kv_heads=2, head_dim=64, num_layers=2)
    fmt = ops.PageFormat(2, 64, 16, 8, 32, torch.bfloat16)
    arena = DevicePageArena(fmt, 60, num_layers=2, max_slots=5, max_tokens=256)
    arena.track_mass()
    model = AttentionStack(spec)
    runner = DeviceRunner(model, arena)
    a, b = arena.open_slot(), arena.open_slot()
    gen = torch.Generator().manual_seed(3)
    runner.execute([a, b], torch.randn((2, 50, 128), generator=gen).cuda().to(torch.bfloat16))
    arena.evict([a, b], [0, 20])

    class Fails:
        spec = model.spec

        def forward(self, *_a, **_k):
            raise RuntimeError("a step that fails")

    with pytest.raises(RuntimeError):
        DeviceRunner(Fails(), arena).execute([a, b], torch.zeros((2, 1, 128), device="cuda", dtype=torch.bfloat16))
    assert arena.lengths[a] == 0 and arena.lengths[b] == 20 and arena.lens[[a, b]].tolist() == [0, 20]
    res = arena.reserve([a, b], [0, 0])
    assert arena.positions(res).tolist() == [50, 50]
    # emptied by truncation, a slot starts anew
    arena.truncate([a, b], [0, 0])
    assert arena.positions(arena.reserve([a, b], [0, 0])).tolist() == [0, 0]


def test_positions_go_on_after_a_cancelled_step():
    import threading

    from pkv.runner import ForwardRequest, PagedRunner
    from test_gpu_device_cache import _setup

    model, cm = _setup("device")
    handles = [cm.create_handle(f"r{i}", key_type="q8_0", value_type="q8_0") for i in range(3)]
    arena = handles[0].bundle.entries[0].arena
    arena.track_mass()
    runner = PagedRunner(model)
    gen = torch.Generator(device="cuda").manual_seed(1)

    def run(widths, cancel):
        return runner.execute([
            ForwardRequest(None, (), h.bundle.entries, phase="prefill", runtime=cm, handle=h, request_id=h.request_id,
                           hidden=torch.randn((n, 256), generator=gen, device="cuda").half(), cancel=c)
            for h, n, c in zip(handles, widths, cancel)])

    run([50, 60, 70], [None] * 3)
    slots = [h.bundle.entries[0].slot for h in handles]
    arena.evict(slots, [0, 20, 0])
    stop = threading.Event()
    forward = model.forward

    def forward_and_cancel(*args, **kw):
        stop.set()
        return forward(*args, **kw)

    model.forward = forward_and_cancel
    run([1, 1, 1], [stop, stop, None])
    model.forward = forward
    assert arena.lens[slots].tolist() == [0, 20, 1] and [arena.lengths[s] for s in slots] == [0, 20, 1]
    assert [h.token_count for h in handles] == [0, 20, 1]
    assert arena.positions(arena.reserve(slots, [0, 0, 0])).tolist() == [50, 60, 71]
