"""GPU: rotation with append of projections that are views of every order, against the same
of dense copies, bit for bit."""

from __future__ import annotations

import pytest

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")


@pytest.fixture(scope="module", autouse=True)
def _gpu():
    if not torch.cuda.is_available():
        pytest.skip("no GPU")


def _views(batch, tokens, width):
    gen = torch.Generator().manual_seed(batch + tokens)
    make = lambda *shape: torch.randn(shape, generator=gen).cuda().bfloat16()
    yield make(tokens, batch, width).transpose(0, 1)
    yield make(batch, tokens + 3, width)[:, -tokens:]
    yield make(batch, tokens, width + 16)[..., 8:8 + width]
    yield make(2 * batch, tokens, width)[::2]
    yield make(batch, width, tokens).transpose(1, 2)
    yield make(1, tokens, width).expand(batch, tokens, width)


@pytest.mark.parametrize("bits", [4, 8, 16])
@pytest.mark.parametrize("batch,tokens", [(1, 1), (5, 1), (200, 1), (1, 7), (4, 3), (3, 60)])
def test_padded_and_packed(bits, batch, tokens):
    from pkv import ops

    fmt = ops.PageFormat(2, 64, 16, bits, 32, torch.bfloat16)
    inv = (10000.0 ** (-torch.arange(32, dtype=torch.float64) / 32)).float().cuda()
    pages = 8
    table = torch.arange(batch * pages, dtype=torch.int32, device="cuda").view(batch, pages)
    starts = torch.arange(batch, dtype=torch.int32, device="cuda") % 40

    def run(x, **kw):
        pool = ops.allocate_pool(fmt, batch * pages)
        out = ops.rope_append(fmt, pool, x, table, starts, inv, 4, with_kv=True, **kw)
        return (*out, pool)

    for x in _views(batch, tokens, 8 * 64):
        dense = torch.empty(x.shape, dtype=x.dtype, device="cuda").copy_(x)
        want = run(dense)
        for a, b in zip(run(x), want):
            assert torch.equal(a.view(torch.uint8), b.view(torch.uint8))
        # the same rows packed: one sequence after the other
        if tokens == 1 or batch == 1:
            rows = x[:, 0] if tokens == 1 else x[0]
            got = run(rows, row_starts=torch.arange(batch + 1, dtype=torch.int32) * tokens)
            assert torch.equal(got[3], want[3])
            for a, b in zip(got[:3], want):
                b = b.transpose(1, 2).reshape(a.shape)
                assert torch.equal(a.view(torch.uint8), b.view(torch.uint8))
