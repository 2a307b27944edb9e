"""CPU: the rows of a projection that the rotation with append reads, as its launch gets
them, for views of every order."""

from __future__ import annotations

import pytest

torch = pytest.importorskip("torch")

HEADS, WIDTH = 2, 6 * 8


def _views(batch, tokens):
    """``(name, [batch, tokens, width] view)`` of fresh memory, each of another order."""
    numbers = lambda *shape: torch.arange(torch.Size(shape).numel()).view(shape).bfloat16()
    yield "dense", numbers(batch, tokens, WIDTH)
    yield "time-major", numbers(tokens, batch, WIDTH).transpose(0, 1)
    yield "last tokens", numbers(batch, tokens + 3, WIDTH)[:, -tokens:]
    yield "first tokens", numbers(batch, tokens + 1, WIDTH)[:, :tokens]
    yield "part of wider rows", numbers(batch, tokens, WIDTH + 16)[..., 8:8 + WIDTH]
    yield "every other sequence", numbers(2 * batch, tokens, WIDTH)[::2]
    yield "every other token", numbers(batch, 2 * tokens, WIDTH)[:, ::2]
    yield "one row for all", numbers(WIDTH).expand(batch, tokens, WIDTH)
    yield "one sequence for all", numbers(1, tokens, WIDTH).expand(batch, tokens, WIDTH)
    yield "columns", numbers(batch, WIDTH, tokens).transpose(1, 2)
    yield "columns of sequences", numbers(WIDTH, batch, tokens).permute(1, 2, 0)
    yield "overlapping", numbers(batch * tokens + WIDTH).as_strided((batch, tokens, WIDTH), (tokens, 1, 1))


class _Launched(Exception):
    pass


@pytest.fixture
def launched(monkeypatch):
    """``ops`` whose launches raise with their arguments, and which takes CPU tensors."""
    from pkv import ops

    def launch(device, what, entry, *args):
        raise _Launched(args)

    monkeypatch.setattr(ops, "_check_float", lambda *a: None)
    monkeypatch.setattr(ops, "_launch", launch)
    kept = []
    plain = torch.Tensor.data_ptr
    monkeypatch.setattr(torch.Tensor, "data_ptr", lambda t: (kept.append(t), plain(t))[1])
    return ops, kept


def _read(ops, kept, qkv, rows, **kw):
    """The rows as the kernel reads them: row i at the address + i * the stride."""
    fmt = ops.PageFormat(2, 8, 16, 16, 32, torch.bfloat16)
    batch = kw.pop("batch")
    with pytest.raises(_Launched) as launch:
        ops.rope_append(fmt, torch.zeros((1, fmt.page_bytes), dtype=torch.uint8), qkv,
                        torch.zeros((batch, 1), dtype=torch.int32), [0] * batch, torch.ones(4), HEADS, **kw)
    _, _, _, at, stride, count, *_ = launch.value.args[0]
    source = next(t for t in kept if torch.Tensor.data_ptr(t) == at and t.dtype is torch.bfloat16)
    assert count == rows
    # (nothing past the memory that the tensor has)
    assert source.storage_offset() + (rows - 1) * stride + WIDTH <= source.untyped_storage().nbytes() // 2
    assert stride >= WIDTH
    return source.as_strided((rows, WIDTH), (stride, 1))


@pytest.mark.parametrize("batch,tokens", [(1, 1), (4, 1), (1, 5), (4, 5), (2, 3)])
def test_padded(launched, batch, tokens):
    ops, kept = launched
    for name, x in _views(batch, tokens):
        kept.clear()
        got = _read(ops, kept, x, batch * tokens, batch=batch)
        assert torch.equal(got, x.reshape(-1, WIDTH)), name


@pytest.mark.parametrize("rows", [1, 2, 7])
def test_packed(launched, rows):
    ops, kept = launched
    views = [(f"{n} sequences: {name}", x[:, 0] if n > 1 else x[0]) for n in (1, rows) for name, x in
             _views(*((1, rows) if n == 1 else (rows, 1)))]
    views.append(("a column", torch.arange(WIDTH).bfloat16()[:, None].t().expand(1, WIDTH)))
    for name, x in views:
        kept.clear()
        got = _read(ops, kept, x, x.shape[0], batch=1, row_starts=[0, x.shape[0]])
        assert torch.equal(got, x), name
