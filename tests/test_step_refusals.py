"""CPU: what the operators of a serving step refuse, before any launch."""

from __future__ import annotations

import pytest

from pkv import _native as nat

torch = pytest.importorskip("torch")

FAKE = 4096   # never dereferenced: the call fails or returns first


def _layout(**kw):
    base = dict(num_kv_heads=8, head_dim=128, page_tokens=16, bits=8, group_size=64, float_kind=0)
    base.update(kw)
    return nat.Layout(*base.values())


def _rope(**kw):
    a = dict(stream=None, layout=_layout(), pool=FAKE, num_pages=10, qkv=FAKE, stride=48 * 128, rows=6, heads=32,
             batch=2, tokens=0, row_starts=FAKE, widths=None, start_pos=FAKE, positions=None, axes=1, inv_freq=FAKE,
             freqs=64, axis=None, table=FAKE, max_pages=4, q=FAKE, k=None, v=None)
    a.update(kw)
    return nat.load().pkv_rope_append(*a.values())


@pytest.mark.parametrize("kw,code", [
    (dict(layout=_layout(bits=5)), 2), (dict(heads=0), 1), (dict(rows=-1), 1), (dict(batch=-1), 1),
    (dict(freqs=65), 1), (dict(freqs=-1), 1), (dict(axes=0), 1), (dict(axes=9), 1), (dict(axis=FAKE), 1),
    (dict(widths=FAKE), 1), (dict(row_starts=None, tokens=2), 1), (dict(stride=48 * 128 - 1), 1),
    (dict(stride=1 << 41), 2), (dict(rows=(1 << 23) + 1), 2), (dict(batch=(1 << 20) + 1), 2),
    (dict(heads=1 << 17, stride=1 << 32), 2), (dict(max_pages=1 << 28), 1), (dict(qkv=None), 1), (dict(q=None), 1),
    (dict(start_pos=None), 1), (dict(inv_freq=None), 1), (dict(pool=None), 1), (dict(table=None), 1),
    (dict(k=FAKE), 1), (dict(v=FAKE), 1)])
def test_rope_append(kw, code):
    assert _rope(**kw) == code and nat.last_error()


def _prompt(**kw):
    a = dict(stream=None, q=FAKE, qs=32 * 128, k=FAKE, ks=8 * 128, v=FAKE, vs=8 * 128, kind=0, rows=6, batch=2,
             row_starts=FAKE, heads=32, kv_heads=8, dim=128, scale=1.0, out=FAKE)
    a.update(kw)
    return nat.load().pkv_prompt_attention(*a.values())


@pytest.mark.parametrize("kw,code", [
    (dict(kind=2), 1), (dict(rows=-1), 1), (dict(batch=-1), 1), (dict(heads=0), 1), (dict(kv_heads=0), 1),
    (dict(heads=30), 1), (dict(dim=0), 1), (dict(dim=264), 2), (dict(dim=100), 2), (dict(scale=float("inf")), 1),
    (dict(qs=32 * 128 - 8), 1), (dict(ks=8 * 127), 1), (dict(vs=1000), 1), (dict(ks=8 * 128 + 4), 1),
    (dict(vs=(1 << 23) + 8), 2), (dict(rows=(1 << 24) + 1), 2), (dict(batch=(1 << 20) + 1), 2),
    (dict(rows=1 << 24), 2), (dict(q=None), 1), (dict(k=None), 1), (dict(v=None), 1), (dict(out=None), 1),
    (dict(row_starts=None), 1), (dict(q=FAKE + 8), 1), (dict(out=FAKE + 2), 1)])
def test_prompt_attention(kw, code):
    assert _prompt(**kw) == code and nat.last_error()


def _shared(**kw):
    a = dict(stream=None, layout=_layout(), pool=FAKE, num_pages=10, queries=FAKE, batch=2, heads=32, nq=1,
             table=FAKE, max_pages=4, lens=FAKE, q_pos=None, widths=None, groups=1, members=FAKE, count=2,
             starts=FAKE, prefix=FAKE, scale=1.0, ws=FAKE, ws_bytes=1 << 40, out=FAKE, zero_others=0)
    a.update(kw)
    return nat.load().pkv_shared_attention(*a.values())


@pytest.mark.parametrize("kw,code", [
    (dict(layout=_layout(bits=5)), 2), (dict(heads=30), 1), (dict(heads=0), 1), (dict(nq=0), 1), (dict(nq=9), 2),
    (dict(nq=5, layout=_layout(head_dim=256)), 2), (dict(batch=-1), 1), (dict(groups=-1), 1), (dict(count=-1), 1),
    (dict(groups=1025), 2), (dict(count=1025), 2), (dict(batch=(1 << 20) + 1), 2), (dict(max_pages=1 << 28), 1),
    (dict(scale=float("nan")), 1), (dict(pool=None), 1), (dict(queries=None), 1), (dict(table=None), 1),
    (dict(lens=None), 1), (dict(members=None), 1), (dict(starts=None), 1), (dict(prefix=None), 1), (dict(out=None), 1),
    (dict(num_pages=0), 1), (dict(max_pages=0), 1), (dict(ws=None), 3), (dict(ws_bytes=100), 3), (dict(ws=FAKE + 8), 1),
    (dict(heads=512, layout=_layout(num_kv_heads=512), count=1024), 2), (dict(batch=1 << 20, nq=2), 2)])
def test_shared_attention(kw, code):
    assert _shared(**kw) == code and nat.last_error()


def test_shared_workspace():
    size = nat.load().pkv_shared_attention_workspace_bytes
    assert size(_layout(), 32, 1, 32, 1) > 0 and size(_layout(), 32, 1, 0, 0) > 0
    assert size(_layout(), 30, 1, 32, 1) == -1 and size(_layout(), 32, 9, 32, 1) == -2


def test_calls_with_nothing_to_do_return():
    assert _shared(batch=0) == 0 and _shared(count=0) == 0 and _shared(groups=0) == 0
    assert _prompt(rows=0) == 0 and _prompt(batch=0) == 0 and _prompt(rows=0, batch=0, q=None, out=None) == 0
    assert _rope(rows=0) == 0 and _rope(batch=0) == 0 and _rope(rows=0, batch=0, qkv=None, q=None) == 0


def test_sections():
    from pkv import ops

    assert ops.rope_axes((2, 3, 1), "cpu").tolist() == [0, 0, 1, 1, 1, 2]
    assert ops.rope_axes((2, 3, 1), "cpu", interleaved=True).tolist() == [0, 1, 2, 0, 1, 1]
    for bad in ((), (1, -1)):
        with pytest.raises(ValueError):
            ops.rope_axes(bad, "cpu")
