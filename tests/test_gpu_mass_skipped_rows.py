"""GPU: attention mass of many sequences of which some have no row: the others' sums are
what they are in a call where every sequence has one."""

from __future__ import annotations

import numpy as np
import pytest

from cache_ops_case import mass64, scale_of

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")


@pytest.fixture(scope="module", autouse=True)
def _gpu():
    if not torch.cuda.is_available():
        pytest.skip("no GPU")


def _shared_pages(fmt, lens, rng, pages=96):
    """Sequences over random pages of one small pool (a page may serve many)."""
    from pkv import ops

    pool = ops.allocate_pool(fmt, pages)
    own = torch.arange(pages, dtype=torch.int32, device="cuda").view(pages, 1)
    shape = (pages, fmt.num_kv_heads, fmt.page_tokens, fmt.head_dim)
    k, v = (torch.from_numpy(rng.standard_normal(shape, np.float32)).cuda().to(fmt.dtype) for _ in range(2))
    zero = torch.zeros(pages, dtype=torch.int32, device="cuda")
    ops.append_quantize(fmt, pool, k, v, own, zero, zero + fmt.page_tokens)
    width = -(-max(lens) // fmt.page_tokens)
    return pool, torch.from_numpy(rng.integers(0, pages, (len(lens), width), np.int32)).cuda()


# (KV heads, queries): scores kept; K read twice
@pytest.mark.parametrize("hk,nq", [(8, 1), (4, 9)])
@pytest.mark.parametrize("skipped", ["even from 64", "tenth", "half", "all from 60 to 140", "from 100 on"])
def test_skipped_rows(hk, nq, skipped):
    """More units than workgroups, so that each goes from one 64 sequences to the next."""
    from pkv import ops

    fmt = ops.PageFormat(hk, 64, 128, 8, 32, torch.bfloat16)
    batch = 200
    rng = np.random.default_rng(hk)
    lens = rng.integers(1000, 8192, batch).tolist()
    lens[150:155] = [0, 1, 0, 5, 0]
    pool, table = _shared_pages(fmt, lens, rng)
    q = torch.from_numpy(rng.standard_normal((batch, hk * 2, nq, 64), np.float32)).cuda().to(fmt.dtype)
    gone = {"even from 64": [b for b in range(64, 96) if b % 2 == 0], "tenth": np.nonzero(rng.random(batch) < 0.1)[0],
            "half": np.nonzero(rng.random(batch) < 0.5)[0], "all from 60 to 140": range(60, 140),
            "from 100 on": range(100, batch)}[skipped]
    place = rng.permutation(batch).astype(np.int32)
    rows = place.copy()
    rows[list(gone)] = np.resize(np.array([-1, batch, -5, 1 << 30], np.int32), len(gone))
    assert len(gone) > 0
    everyone = torch.full((batch, hk, 8192), -7.0, device="cuda")
    some = everyone.clone()
    kw = dict(scale=scale_of(fmt))
    ops.attention_mass(fmt, pool, q, table, lens, rows=torch.from_numpy(place), out=everyone, **kw)
    ops.attention_mass(fmt, pool, q, table, lens, rows=torch.from_numpy(rows), out=some, **kw)
    live = sorted(set(range(batch)) - set(int(b) for b in gone))
    assert torch.equal(some[place[live]], everyone[place[live]])
    assert (some[place[list(gone)]] == -7.0).all()
    for b in live[::17]:
        want, bound = mass64(fmt, pool, table[b:b + 1], lens[b:b + 1], q[b:b + 1], kw["scale"])
        off = np.abs(some[place[b], :, :lens[b]].double().cpu().numpy() - want[0])
        assert np.all(off <= bound[0]), b
