"""CPU: what the operators on cached state refuse, before any launch."""

from __future__ import annotations

import ctypes

import pytest

from pkv import _native as nat
from pkv.cache_errors import CacheCapacityError
from pkv.modes import ModelCapabilityUnsupported

torch = pytest.importorskip("torch")

FAKE = 4096   # never dereferenced: the call fails or returns first


def _layout(**kw):
    base = dict(num_kv_heads=8, head_dim=128, page_tokens=16, bits=8, group_size=64, float_kind=0)
    base.update(kw)
    return nat.Layout(*base.values())


def _mass(**kw):
    a = dict(stream=None, layout=_layout(), pool=FAKE, num_pages=10, queries=FAKE, batch=2, heads=32, nq=1,
             table=FAKE, max_pages=4, lens=FAKE, q_pos=None, widths=None, scale=1.0, mass=None, counted=None,
             rows=None, mass_rows=2, width=64, ws=FAKE, ws_bytes=1 << 40, out=FAKE)
    a.update(kw)
    return nat.load().pkv_attention_mass(*a.values())


@pytest.mark.parametrize("kw,code", [
    (dict(layout=_layout(bits=5)), 2), (dict(layout=_layout(head_dim=300)), 2), (dict(heads=30), 1), (dict(heads=0), 1),
    (dict(nq=-1), 1), (dict(batch=-1), 1), (dict(max_pages=-1), 1), (dict(scale=float("nan")), 1),
    (dict(scale=float("inf")), 1), (dict(mass_rows=1), 1), (dict(width=-1), 1), (dict(out=None), 1),
    (dict(pool=None), 1), (dict(queries=None), 1), (dict(table=None), 1), (dict(lens=None), 1),
    (dict(nq=1 << 23), 2), (dict(max_pages=1 << 28), 1), (dict(batch=10000, mass_rows=10000), 2),
    (dict(ws=None), 3), (dict(ws_bytes=0), 3), (dict(nq=1 << 20, batch=1000, mass_rows=1000), 2)])
def test_attention_mass(kw, code):
    assert _mass(**kw) == code and nat.last_error()


def test_calls_with_nothing_to_do_return():
    assert _mass(batch=0) == 0 and _mass(max_pages=0) == 0 and _mass(width=0) == 0
    assert _select(batch=0) == 0 and _select(layers=0) == 0
    assert _pages(batch=0) == 0 and _pages(max_keep=0) == 0 and _pages(num_pools=0) == 0
    assert _beam(groups=0) == 0
    assert _rows(count=0) == 0 and _rows(outer=0) == 0 and _rows(row_bytes=0) == 0
    assert _arena(count=0) == 0


def _select(**kw):
    a = dict(stream=None, mass=FAKE, layers=1, mass_rows=2, hk=2, width=100, rows=None, lens=FAKE, batch=2, keep=None,
             max_keep=10, sinks=1, recent=1, kept=FAKE, new_lens=FAKE, new_mass=None, new_width=0)
    a.update(kw)
    return nat.load().pkv_evict_select(*a.values())


@pytest.mark.parametrize("kw,code", [
    (dict(mass_rows=1), 1), (dict(hk=0), 1), (dict(width=1 << 31), 1), (dict(max_keep=-1), 1), (dict(sinks=-1), 1),
    (dict(recent=-1), 1), (dict(new_mass=FAKE, new_width=9), 1), (dict(mass=None), 1), (dict(kept=None), 1),
    (dict(new_lens=None), 1), (dict(lens=None), 1), (dict(layers=1 << 20, hk=1 << 20), 2)])
def test_evict_select(kw, code):
    assert _select(**kw) == code


def _pages(**kw):
    pools = (ctypes.c_void_p * 2)(FAKE, FAKE)
    a = dict(stream=None, layout=_layout(), pools=pools, num_pools=2, num_pages=10, kept=FAKE, new_lens=FAKE, batch=2,
             max_keep=10, src=FAKE, src_pages=4, dst=FAKE, dst_pages=1)
    a.update(kw)
    return nat.load().pkv_evict_pages(*a.values())


@pytest.mark.parametrize("kw,code", [
    (dict(layout=_layout(bits=3)), 2), (dict(num_pools=129), 1), (dict(num_pools=-1), 1), (dict(max_keep=-1), 1),
    (dict(src_pages=1 << 28), 1), (dict(kept=None), 1), (dict(src=None), 1), (dict(dst=None), 1),
    (dict(pools=(ctypes.c_void_p * 2)(FAKE, None)), 1), (dict(batch=10000), 2)])
def test_evict_pages(kw, code):
    assert _pages(**kw) == code


def _beam(**kw):
    a = dict(stream=None, logits=FAKE, kind=0, groups=1, beams=2, vocab=10, gs=20, bs=10, scores=FAKE, done=None,
             pad=0, count=4, ws=FAKE, ws_bytes=1 << 40, out=FAKE, parents=FAKE, tokens=FAKE)
    a.update(kw)
    return nat.load().pkv_beam_select(*a.values())


@pytest.mark.parametrize("kw,code", [
    (dict(kind=3), 1), (dict(beams=0), 1), (dict(beams=65), 2), (dict(vocab=0), 1), (dict(count=0), 1),
    (dict(count=65, vocab=100), 2), (dict(count=21), 1), (dict(vocab=1 << 30, beams=64), 2),
    (dict(groups=1 << 20, vocab=1 << 24), 2), (dict(groups=1 << 24), 2), (dict(gs=-1), 1),
    (dict(done=FAKE, pad=10), 1), (dict(done=FAKE, pad=-1), 1), (dict(scores=None), 1), (dict(tokens=None), 1),
    (dict(ws=None), 3), (dict(ws_bytes=8), 3)])
def test_beam_select(kw, code):
    assert _beam(**kw) == code


def _rows(**kw):
    a = dict(stream=None, state=FAKE, outer=1, num_rows=4, row_bytes=10, targets=FAKE, sources=FAKE, count=2)
    a.update(kw)
    return nat.load().pkv_reorder_rows(*a.values())


@pytest.mark.parametrize("kw,code", [
    (dict(outer=-1), 1), (dict(row_bytes=-1), 1), (dict(count=-1), 1), (dict(count=8193), 2), (dict(outer=65536), 2),
    (dict(row_bytes=(1 << 31) + 1), 2), (dict(state=None), 1), (dict(targets=None), 1)])
def test_reorder_rows(kw, code):
    assert _rows(**kw) == code


def _arena(**kw):
    a = dict(stream=None, state=FAKE, capacity=10, page=16, table=FAKE, num_slots=4, max_pages=8, lens=FAKE,
             slots=FAKE, sources=FAKE, count=2, ws=FAKE, ws_bytes=1 << 40)
    a.update(kw)
    return nat.load().pkv_arena_reorder(*a.values())


@pytest.mark.parametrize("kw,code", [
    (dict(capacity=0), 1), (dict(page=24), 1), (dict(num_slots=0), 1), (dict(max_pages=0), 1), (dict(count=-1), 1),
    (dict(count=4097), 2), (dict(state=None), 1), (dict(sources=None), 1), (dict(ws=None), 3), (dict(ws_bytes=4), 3)])
def test_arena_reorder(kw, code):
    assert _arena(**kw) == code


def test_grids_that_no_launch_takes_and_misaligned_workspaces():
    assert _mass(nq=1 << 16, batch=300, mass_rows=300) == 2 and _mass(ws=FAKE + 8) == 1
    assert _select(layers=1 << 12, hk=1 << 9) == 2
    assert _pages(max_keep=(1 << 29) + 1) == 2
    assert _beam(groups=(1 << 21) + 1, beams=1) == 2 and _beam(groups=1 << 21, beams=3) == 2
    assert _beam(groups=1 << 16, vocab=1 << 20) == 2 and _beam(ws=FAKE + 4) == 1
    assert _rows(row_bytes=1 << 31, count=65) == 2
    assert _arena(max_pages=(1 << 23) + 1) == 2 and _arena(ws=FAKE + 4) == 1


def test_workspace_sizes():
    lib = nat.load()
    assert lib.pkv_attention_mass_workspace_bytes(_layout(), 32, 1, 2, 4) > 0
    assert lib.pkv_attention_mass_workspace_bytes(_layout(), 30, 1, 2, 4) == -1
    assert lib.pkv_beam_workspace_bytes(1, 2, 10, 4) > 0
    assert lib.pkv_beam_workspace_bytes(1, 2, 100, 65) == -2
    assert lib.pkv_beam_workspace_bytes(1, 2, 10, 0) == -1
    assert lib.pkv_arena_reorder_workspace_bytes(2, 8) > 0
    assert lib.pkv_arena_reorder_workspace_bytes(4097, 8) == -2
    assert lib.pkv_arena_reorder_workspace_bytes(-1, 8) == -1


def test_python_checks():
    from pkv import ops

    with pytest.raises(ValueError):
        ops.evict_select(torch.zeros((2, 3)), [1], 1)
    with pytest.raises(ValueError):
        ops.evict_select(torch.zeros((1, 2, 3)), [1], 1)             # not on a device
    with pytest.raises(ValueError):
        ops.beam_select(torch.zeros((1, 2, 3)), torch.zeros((1, 2)), 1)
    with pytest.raises(ValueError):
        ops.beam_select(torch.zeros((1, 2)), torch.zeros((1, 2)), 1)
    with pytest.raises(ValueError):
        ops.reorder_rows(torch.zeros((2, 3)), [0], [1])
    fmt = ops.PageFormat(1, 64, 16, 8, 32, torch.bfloat16)
    with pytest.raises(ValueError):
        ops.attention_mass(fmt, torch.zeros((1, fmt.page_bytes), dtype=torch.uint8),
                           torch.zeros((1, 4, 1, 64), dtype=torch.bfloat16), [[0]], [1], scale=1.0)
    for code, kind in ((1, ValueError), (2, ModelCapabilityUnsupported), (3, CacheCapacityError)):
        with pytest.raises(kind):
            nat.check(code, "call")
