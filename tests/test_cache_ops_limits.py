"""CPU: sizes next to 2^31, where the operators' 32-bit token numbers would end, are
refused before any launch, and the ones below are taken."""

from __future__ import annotations

import pytest

from test_cache_ops_refusals import _beam, _layout, _mass, _select

from pkv import _native as nat

pytest.importorskip("torch")

LAST = (1 << 31) - 1


@pytest.mark.parametrize("kw", [dict(width=LAST), dict(width=LAST - (1 << 15)), dict(max_keep=LAST),
                                dict(max_keep=LAST - 1023), dict(width=LAST, rows=4096, mass_rows=1)])
def test_evict_select(kw):
    assert _select(**kw) == 2 and "tokens" in nat.last_error()


@pytest.mark.parametrize("kind", [0, 1, 2])
@pytest.mark.parametrize("beams,vocab", [(1, LAST), (1, LAST - (1 << 14))])
def test_beam_select(beams, vocab, kind):
    assert _beam(beams=beams, vocab=vocab, kind=kind) == 2 and "pairs" in nat.last_error()
    assert nat.load().pkv_beam_workspace_bytes(1, beams, vocab, 4) == -2
    assert nat.load().pkv_beam_workspace_bytes(1, 1, LAST - (1 << 15), 4) > 0
    assert nat.load().pkv_beam_workspace_bytes(1, 2, (1 << 30) - 1, 4) > 0


@pytest.mark.parametrize("page,pages", [(16, (1 << 27) - 1), (128, (1 << 24) - 1), (64, (1 << 25) - 1)])
@pytest.mark.parametrize("nq", [1, 40])
def test_attention_mass(page, pages, nq):
    layout = _layout(page_tokens=page, num_kv_heads=1)
    kw = dict(layout=layout, max_pages=pages, batch=1, nq=nq)
    assert _mass(**kw) == 2 and "tokens" in nat.last_error()
    size = nat.load().pkv_attention_mass_workspace_bytes
    assert size(layout, 32, nq, 1, pages) == -2
    assert size(layout, 32, nq, 1, (1 << 31) // page - 1024 // page) > 0
