"""Functional layer over libpkv: torch device tensors in and out.

These are the primitives the reference-named classes (``pkv.arena``,
``pkv.paged``, ``pkv.paged_attention``) are built on.  Every function enqueues
HIP work on the current torch stream through the C ABI and never falls back to
a CPU implementation.
"""

from __future__ import annotations

import math
from dataclasses import dataclass
from functools import cached_property

import torch

from pkv import _native as nat

FLOAT_KINDS = {torch.bfloat16: 0, torch.float16: 1}
DTYPES = {0: torch.bfloat16, 1: torch.float16}


@dataclass(frozen=True)
class PageFormat:
    """One layer's page layout; the C ``pkv_layout`` plus derived sizes.

    ``bits`` is 4 or 8 for affine-quantized pages and 16 for float pages
    (the reference's ``BlockLayout.quantization_bits`` None).
    """

    num_kv_heads: int
    head_dim: int
    page_tokens: int
    bits: int = 16
    group_size: int = 32
    dtype: torch.dtype = torch.bfloat16

    def __post_init__(self):
        if self.dtype not in FLOAT_KINDS:
            from pkv.modes import ModelCapabilityUnsupported

            raise ModelCapabilityUnsupported("unsupported paged storage precision")
        if self.page_bytes < 0:
            nat.check(nat.PKV_UNSUPPORTED, "page layout")

    # (computed once per format: every call passes them)
    @cached_property
    def c_layout(self):
        return nat.Layout(self.num_kv_heads, self.head_dim, self.page_tokens, self.bits,
                          self.group_size if self.bits != 16 else 32, FLOAT_KINDS[self.dtype])

    @cached_property
    def page_bytes(self):
        return int(nat.load().pkv_page_bytes(self.c_layout))

    @cached_property
    def stored_dim(self):
        return int(nat.load().pkv_stored_dim(self.c_layout))

    @property
    def quantized(self):
        return self.bits != 16

    @property
    def reference_dim(self):
        """Padded head dim of the reference format (``paged.py:31``)."""
        if not self.quantized:
            return self.head_dim
        return (self.head_dim + self.group_size - 1) // self.group_size * self.group_size


def allocate_pool(fmt: PageFormat, num_pages: int, device="cuda"):
    """Device page pool ``[num_pages, page_bytes]`` uint8 (zeroed)."""
    return torch.zeros((num_pages, fmt.page_bytes), dtype=torch.uint8, device=device)


def _i32(x, device):
    if x is None:
        return None
    if isinstance(x, torch.Tensor):
        if x.dtype is torch.int32 and x.device == device and x.is_contiguous():
            return x
        t = x.to(device=device, dtype=torch.int32)
    else:
        t = torch.as_tensor(x, dtype=torch.int32).to(device)
    return t.contiguous()


def _check_float(t, fmt, name):
    if t.dtype != fmt.dtype:
        raise ValueError(f"{name} dtype {t.dtype} differs from the page dtype {fmt.dtype}")
    if not t.is_cuda:
        raise ValueError(f"{name} must be a device tensor")


def append_quantize(fmt: PageFormat, pool, keys, values, block_table, start_pos, widths=None,
                    new_lens=None):
    """Write ``keys/values [B, HK, T, D]`` at positions ``start_pos[b] + t``."""
    if keys.shape != values.shape or keys.dim() != 4:
        raise ValueError("paged append requires matching [B, HK, T, D] K/V tensors")
    batch, heads, tokens, dim = keys.shape
    if heads != fmt.num_kv_heads or dim != fmt.head_dim:
        raise ValueError("paged append layout mismatch")
    _check_float(keys, fmt, "keys")
    _check_float(values, fmt, "values")
    device = keys.device
    table = _i32(block_table, device)
    if table.dim() != 2 or table.shape[0] != batch:
        raise ValueError("block table must be [batch, max_pages]")
    start = _i32(start_pos, device)
    width = _i32(widths, device)
    keys, values = keys.contiguous(), values.contiguous()
    code = nat.load().pkv_append_quantize(
        nat.stream_handle(device), fmt.c_layout, nat.ptr(pool), pool.shape[0], nat.ptr(keys),
        nat.ptr(values), batch, tokens, nat.ptr(table), table.shape[1], nat.ptr(start),
        nat.ptr(width), nat.ptr(new_lens))
    nat.check(code, "paged append")


def attention_waves(fmt: PageFormat, num_heads, num_queries):
    """Waves the attention kernel keeps resident for this shape (the default grid)."""
    waves = int(nat.load().pkv_attention_waves(fmt.c_layout, num_heads, num_queries))
    if waves <= 0:
        nat.check(nat.PKV_LAUNCH_FAILED, "attention waves")
    return waves


DECODE_KERNELS = {"mfma": 0, "valu": 1}


def select_decode_kernel(kind):
    """Choose the kernel for decode rows (at most 4 query rows per KV head over
    quantized pages, head_dim <= 128): ``"mfma"`` (the default) or ``"valu"``
    (the same split and merge with vector-ALU dot products).  Process-wide;
    returns the previous choice."""
    if kind not in DECODE_KERNELS:
        raise ValueError(f"decode kernel must be one of {sorted(DECODE_KERNELS)}")
    previous = int(nat.load().pkv_select_decode_kernel(DECODE_KERNELS[kind]))
    if previous < 0:
        nat.check(previous, "select decode kernel")
    return {v: k for k, v in DECODE_KERNELS.items()}[previous]


def default_waves(fmt: PageFormat, num_heads, num_queries, batch):
    """The waves ``paged_attention`` uses by default for this shape and batch."""
    waves = int(nat.load().pkv_attention_default_waves(fmt.c_layout, num_heads, num_queries,
                                                         batch))
    if waves <= 0:
        nat.check(nat.PKV_LAUNCH_FAILED, "attention waves")
    return waves


def decode_queries(fmt: PageFormat, num_heads, num_queries):
    """Queries per sequence of the split-K decode part of a call: all of them
    when the decode kernel serves the call (at most 32 query rows per KV head,
    16 at head_dim > 128), else the most a mixed batch's narrow sequences may
    have there (0 when the GQA ratio leaves none)."""
    gqa = num_heads // fmt.num_kv_heads
    limit = 16 if fmt.stored_dim > 128 else 32
    return num_queries if num_queries * gqa <= limit else limit // max(gqa, 1)


def workspace_bytes(fmt: PageFormat, num_heads, num_queries, waves):
    return int(nat.load().pkv_attention_workspace_bytes(fmt.c_layout, num_heads, num_queries,
                                                          waves))


# (waves, workspace bytes, wide) of a call shape with default waves: a few integers
# per format, heads, queries, batch, device and decode kernel, as the library
# computed them (cleared when it holds many shapes).
_PLANS = {}
_MAX_PLANS = 4096


def _plan(fmt, heads, nq, batch, device):
    """The default waves of a call, the workspace it runs best with and whether
    it is wide, the same whichever entry point asks first."""
    key = (fmt, heads, nq, batch, device, nat.load().decode_kernel.value)
    plan = _PLANS.get(key)
    if plan is None:
        waves = default_waves(fmt, heads, decode_queries(fmt, heads, nq) or nq, batch)
        plan = (waves, call_workspace_bytes(fmt, heads, nq, batch, waves), is_wide(fmt, heads, nq))
        if len(_PLANS) >= _MAX_PLANS:
            _PLANS.clear()
        _PLANS[key] = plan
    return plan


def split_waves(fmt, heads, nq, batch, device):
    """The default waves, to be passed explicitly: the call then always runs the
    equal split over them, whatever its block table's width -- the arenas' calls
    give the same bits from host tables (as wide as the batch) and from the
    device's (as wide as ``max_tokens``)."""
    return _plan(fmt, heads, nq, batch, device)[0]


def is_wide(fmt, heads, nq):
    """Whether the prefill kernel serves a call's query blocks (more rows per KV
    head than the decode kernel takes)."""
    return decode_queries(fmt, heads, nq) != nq


def call_workspace_bytes(fmt, heads, nq, batch, waves):
    """Workspace with which a call of ``batch`` sequences runs best (and which
    the calls below take when given none): ``workspace_bytes``, and for a wide
    call the partials of cut prefill spans as well."""
    if is_wide(fmt, heads, nq):
        need = int(nat.load().pkv_attention_batch_workspace_bytes(fmt.c_layout, heads, nq, batch,
                                                                  waves))
    else:
        need = workspace_bytes(fmt, heads, nq, waves)
    if need < 0:
        nat.check(nat.PKV_INVALID_ARGUMENT, "paged attention workspace")
    return need


# One attention workspace per device, grown on demand; calls on one stream
# share it (each call's partials are merged before the next call starts).
_WORKSPACES = {}


def attention_workspace(device, nbytes):
    """A workspace of at least ``nbytes`` on ``device`` (cached, grown on demand)."""
    key = device if isinstance(device, torch.device) else torch.device(device)
    ws = _WORKSPACES.get(key)
    if ws is None or ws.numel() < nbytes:
        ws = torch.empty(max(int(nbytes), 256), dtype=torch.uint8, device=key)
        _WORKSPACES[key] = ws
    return ws


def _wide_workspace(device, nbytes, least):
    """The workspace of a wide call that was given none: the stream's own memory
    of exactly that size -- wide calls on other streams or threads may overlap
    it, and whether spans are cut (and so the output's bits) must not depend on
    what grew the shared one.  Without room for it, ``least()`` bytes, with
    which the call runs whole spans."""
    try:
        return torch.empty(max(nbytes, 256), dtype=torch.uint8, device=device)
    except torch.OutOfMemoryError:
        return torch.empty(max(least(), 256), dtype=torch.uint8, device=device)


def paged_attention(fmt: PageFormat, pool, queries, block_table, seq_lens, *, scale, q_pos=None,
                    widths=None, waves=0, workspace=None, out=None):
    """Attention of ``queries [B, H, Q, D]`` over the paged cache.

    ``seq_lens`` counts the tokens in each sequence's cache (after the
    append) and stays on the device: the decode kernel shares the tiles of
    all sequences out over ``waves`` waves (default 0: ``default_waves``, or
    the library's form for short block tables and few segments);
    query blocks past 32 rows per KV head run on the prefill kernel -- and
    in a mixed batch (``widths`` given), the sequences narrow enough for the
    decode kernel still go to it, in the same call (``waves`` then sizes that
    part).  ``workspace`` (bytes from ``workspace_bytes``) may be given by the
    caller.
    """
    if queries.dim() != 4:
        raise ValueError("queries must be [B, H, Q, D]")
    batch, heads, nq, dim = queries.shape
    if dim != fmt.head_dim:
        raise ValueError("query head dimension differs from the page layout")
    _check_float(queries, fmt, "queries")
    device = queries.device
    table = _i32(block_table, device)
    lens = _i32(seq_lens, device)
    if waves <= 0:
        waves, need, wide = _plan(fmt, heads, nq, batch, device)
        if not wide:
            waves = 0  # the library's choice, within the workspace of its default waves
    else:
        need, wide = call_workspace_bytes(fmt, heads, nq, batch, waves), is_wide(fmt, heads, nq)
    if workspace is None:
        workspace = (_wide_workspace(device, need, lambda: workspace_bytes(fmt, heads, nq, waves))
                     if wide else attention_workspace(device, need))
    elif workspace.device != device or workspace.dtype != torch.uint8 or \
            not workspace.is_contiguous():
        raise ValueError("attention workspace must be a contiguous uint8 tensor on the "
                         "queries' device")
    # the kernels read queries and write out as dense [B, H, Q, D]
    queries = queries.contiguous()
    if out is None:
        out = torch.empty(queries.shape, dtype=queries.dtype, device=device)
    elif (tuple(out.shape) != tuple(queries.shape) or out.dtype != queries.dtype
          or out.device != device or not out.is_contiguous()):
        raise ValueError("out must be a contiguous tensor of the queries' shape, dtype and "
                         "device")
    code = nat.load().pkv_paged_attention(
        nat.stream_handle(device), fmt.c_layout, nat.ptr(pool), pool.shape[0], nat.ptr(queries),
        batch, heads, nq, nat.ptr(table), table.shape[1], nat.ptr(lens),
        nat.ptr(_i32(q_pos, device)), nat.ptr(_i32(widths, device)), float(scale),
        int(waves), nat.ptr(workspace), workspace.numel(), nat.ptr(out))
    nat.check(code, "paged attention")
    return out


def append_paged_attention(fmt: PageFormat, pool, keys, values, queries, block_table, seq_lens, *,
                           scale, waves=0, workspace=None, out=None):
    """One single-token step: append ``keys``/``values [B, HK, 1, D]`` at
    position ``seq_lens - 1`` (``seq_lens`` counts the tokens after the
    append) and attend ``queries [B, H, 1, D]`` -- one launch where the decode
    kernel serves the shape (at most 8 query rows per KV head), else an
    append launch and the attention.  Pages equal ``append_quantize``'s bit
    for bit, outputs ``paged_attention``'s within its rounding (its split may
    cut the tiles elsewhere)."""
    if queries.dim() != 4 or queries.shape[2] != 1:
        raise ValueError("queries must be [B, H, 1, D]")
    batch, heads, _, dim = queries.shape
    shape = (batch, fmt.num_kv_heads, 1, dim)
    if dim != fmt.head_dim or tuple(keys.shape) != shape or tuple(values.shape) != shape:
        raise ValueError(f"keys and values must be {shape} and the queries' head dimension "
                         "the page layout's")
    for name, t in (("queries", queries), ("keys", keys), ("values", values)):
        _check_float(t, fmt, name)
    device = queries.device
    table = _i32(block_table, device)
    lens = _i32(seq_lens, device)
    if waves <= 0:
        waves, (_, need, wide) = 0, _plan(fmt, heads, 1, batch, device)
    else:
        need, wide = call_workspace_bytes(fmt, heads, 1, batch, waves), is_wide(fmt, heads, 1)
    if workspace is None:
        workspace = (_wide_workspace(device, need, lambda: 0) if wide
                     else attention_workspace(device, need))
    elif workspace.device != device or workspace.dtype != torch.uint8 or \
            not workspace.is_contiguous():
        raise ValueError("attention workspace must be a contiguous uint8 tensor on the "
                         "queries' device")
    queries, keys, values = queries.contiguous(), keys.contiguous(), values.contiguous()
    if out is None:
        out = torch.empty(queries.shape, dtype=queries.dtype, device=device)
    elif (tuple(out.shape) != tuple(queries.shape) or out.dtype != queries.dtype
          or out.device != device or not out.is_contiguous()):
        raise ValueError("out must be a contiguous tensor of the queries' shape, dtype and "
                         "device")
    code = nat.load().pkv_append_paged_attention(
        nat.stream_handle(device), fmt.c_layout, nat.ptr(pool), pool.shape[0], nat.ptr(keys),
        nat.ptr(values), nat.ptr(queries), batch, heads, nat.ptr(table), table.shape[1],
        nat.ptr(lens), float(scale), int(waves), nat.ptr(workspace), workspace.numel(),
        nat.ptr(out))
    nat.check(code, "append + paged attention")
    return out


def gather_pages(fmt: PageFormat, pool, page_ids):
    """Pages in the reference's per-page tensor format (``paged_attention.py:31-35``).

    Quantized: ``(k_codes [N,HK,P,Dq] u8, k_scale [N,HK,P,Dp/G] f16, k_bias,
    v_codes, v_scale, v_bias)``; float: ``(k [N,HK,P,D], v)``.
    """
    ids = _i32(page_ids, pool.device)
    n = ids.numel()
    shape = (n, fmt.num_kv_heads, fmt.page_tokens)
    if fmt.quantized:
        dq = fmt.reference_dim * fmt.bits // 8
        ng = fmt.reference_dim // fmt.group_size
        kc = torch.empty(shape + (dq,), dtype=torch.uint8, device=pool.device)
        vc = torch.empty_like(kc)
        ks, kb, vs, vb = (torch.empty(shape + (ng,), dtype=torch.float16, device=pool.device)
                          for _ in range(4))
        outs = (kc, ks, kb, vc, vs, vb)
    else:
        k = torch.empty(shape + (fmt.head_dim,), dtype=fmt.dtype, device=pool.device)
        v = torch.empty_like(k)
        outs = (k, None, None, v, None, None)
    code = nat.load().pkv_gather_pages(nat.stream_handle(pool.device), fmt.c_layout,
                                       nat.ptr(pool), pool.shape[0], nat.ptr(ids), n,
                                       *[nat.ptr(t) for t in outs])
    nat.check(code, "page gather")
    return outs if fmt.quantized else (outs[0], outs[3])


def copy_pages(fmt: PageFormat, pool, src_ids, dst_ids):
    src = _i32(src_ids, pool.device)
    dst = _i32(dst_ids, pool.device)
    if src.numel() != dst.numel():
        raise ValueError("page copy requires matching id lists")
    code = nat.load().pkv_copy_pages(nat.stream_handle(pool.device), fmt.c_layout, nat.ptr(pool),
                                     pool.shape[0], nat.ptr(src), nat.ptr(dst), src.numel())
    nat.check(code, "page copy")


def quantize_rows(values, bits, group_size=32):
    """Reference ``quantize_page`` over the last axis: ``(codes, scale f16, bias f16)``."""
    if values.dtype not in FLOAT_KINDS:
        raise ValueError("quantize expects float16 or bfloat16 values")
    values = values.contiguous()
    dim = values.shape[-1]
    rows = values.numel() // dim if dim else 0
    padded = (dim + group_size - 1) // group_size * group_size
    lead = tuple(values.shape[:-1])
    codes = torch.empty(lead + (padded * bits // 8,), dtype=torch.uint8, device=values.device)
    scale = torch.empty(lead + (padded // group_size,), dtype=torch.float16, device=values.device)
    bias = torch.empty_like(scale)
    code = nat.load().pkv_quantize_rows(nat.stream_handle(values.device), nat.ptr(values), rows,
                                        dim, bits, group_size, FLOAT_KINDS[values.dtype],
                                        nat.ptr(codes), nat.ptr(scale), nat.ptr(bias))
    nat.check(code, "quantize")
    return codes, scale, bias


def dequantize_rows(state, bits, dim, group_size=32):
    """Reference ``dequantize_page``: float32 ``[..., dim]``."""
    codes, scale, bias = (t.contiguous() for t in state)
    rows = scale.numel() // scale.shape[-1] if scale.dim() else 0
    out = torch.empty(tuple(codes.shape[:-1]) + (dim,), dtype=torch.float32, device=codes.device)
    code = nat.load().pkv_dequantize_rows(nat.stream_handle(codes.device), nat.ptr(codes),
                                          nat.ptr(scale), nat.ptr(bias), rows, dim, bits,
                                          group_size, nat.ptr(out))
    nat.check(code, "dequantize")
    return out


_FLOAT_KIND = {torch.bfloat16: 0, torch.float16: 1}


def rope_qkv(qkv, positions, inv_freq, heads, kv_heads):
    """Rotate-half RoPE of a fused projection ``qkv [B, T, (heads + 2*kv_heads) * D]``
    at ``positions [B, T]``: returns ``q [B, heads, T, D]``, ``k, v [B, kv_heads, T, D]``
    (q and k rotated, v copied), contiguous, in ``qkv``'s dtype.  Float32 math as
    the reference's ``apply_rope`` (``models/shared/transformer.py:32-90``)."""
    if qkv.dim() != 3 or qkv.dtype not in _FLOAT_KIND or not qkv.is_cuda:
        raise ValueError("qkv must be a [B, T, width] f16/bf16 device tensor")
    batch, tokens, width = qkv.shape
    if width % (heads + 2 * kv_heads):
        raise ValueError("qkv width is not (heads + 2*kv_heads) * head_dim")
    dim = width // (heads + 2 * kv_heads)
    if dim % 2 or dim > 256 or inv_freq.numel() != dim // 2:
        raise ValueError("RoPE needs an even head dimension <= 256 and dim/2 frequencies")
    if tuple(positions.shape) != (batch, tokens):
        raise ValueError("positions must be [B, T]")
    device = qkv.device
    qkv = qkv.contiguous()
    pos = _i32(positions, device)
    inv = inv_freq.to(device=device, dtype=torch.float32).contiguous()
    q = torch.empty((batch, heads, tokens, dim), dtype=qkv.dtype, device=device)
    k = torch.empty((batch, kv_heads, tokens, dim), dtype=qkv.dtype, device=device)
    v = torch.empty_like(k)
    code = nat.load().pkv_rope_qkv(nat.stream_handle(device), nat.ptr(qkv), batch, tokens, heads,
                                   kv_heads, dim, _FLOAT_KIND[qkv.dtype], nat.ptr(pos),
                                   nat.ptr(inv), nat.ptr(q), nat.ptr(k), nat.ptr(v))
    nat.check(code, "rope")
    return q, k, v



# ---- which cached state lives on ---------------------------------------------------


def _launch(device, what, entry, *args):
    """Call a C entry point on the current stream of ``device``, as its current device."""
    index, current = device.index, torch._C._cuda_getDevice()
    if current == index:
        code = entry(torch._C._cuda_getCurrentRawStream(index), *args)
    else:
        torch._C._cuda_setDevice(index)
        try:
            code = entry(torch._C._cuda_getCurrentRawStream(index), *args)
        finally:
            torch._C._cuda_setDevice(current)
    if code:
        nat.check(code, what)


def _dense(t, dtype, device, dims):
    return (isinstance(t, torch.Tensor) and t.dtype is dtype and t.device == device
            and t.dim() == dims and t.is_contiguous())


def _check_dense(t, dtype, device, name, dims):
    if not _dense(t, dtype, device, dims):
        raise ValueError(f"{name} must be a contiguous {dims}-dimensional {dtype} tensor on {device}")


def _per_row(x, device, count, name):
    """An int32 operand of ``count`` values on the device."""
    t = _i32(x, device)
    if t.numel() != count:
        raise ValueError(f"{name} must hold {count} values")
    return t


def _distinct(x, name):
    """Refuse a host list that names a row twice (a tensor is the caller's to know)."""
    if x is not None and not isinstance(x, torch.Tensor):
        named = [int(v) for v in x if v >= 0]
        if len(set(named)) != len(named):
            raise ValueError(f"{name} must be distinct")


def _address(x, device, count, name):
    """``(tensor, its address)`` of an int32 operand of ``count`` values; None: NULL."""
    if x is None:
        return None, None
    t = _per_row(x, device, count, name)
    return t, t.data_ptr()


def _int32(value, name):
    """A number for a 32-bit argument (ctypes would drop what lies above)."""
    if not -2 ** 31 <= value < 2 ** 31:
        raise ValueError(f"{name} does not fit 32 bits")
    return value


def _scratch(nbytes, device, what, given=None):
    """The caller's workspace, or the stream's own memory of that size."""
    if nbytes < 0:
        nat.check(-nbytes, what)
    if given is None:
        return torch.empty(nbytes or 16, dtype=torch.uint8, device=device)
    if given.device != device or given.dtype is not torch.uint8 or not given.is_contiguous():
        raise ValueError(f"{what} workspace must be a contiguous uint8 tensor on {device}")
    return given


def attention_mass(fmt: PageFormat, pool, queries, block_table, seq_lens, *, scale, q_pos=None,
                   widths=None, mass=None, counted=None, rows=None, workspace=None, out=None):
    """Attention weight of ``queries [B, H, Q, D]`` on every cached token, summed over
    the query rows of each KV head and added to the sums so far.

    ``mass [R, HK, N]`` (float32) holds the sums so far (None: zeros) in rows
    ``rows [B]`` (default: row b; distinct), of which the first ``counted[b]``
    tokens of sequence b are read (default: all).  The new sums go to ``out``
    (default: ``mass`` in place, or new zeros ``[B, HK, pages * page_tokens]``),
    which is returned; its entries from ``seq_lens[b]`` on, and rows that no
    sequence of the call has, are left as they are.  The other operands are
    ``paged_attention``'s; a query that sees no token adds nothing.
    """
    if queries.dim() != 4:
        raise ValueError("queries must be [B, H, Q, D]")
    batch, heads, nq, dim = queries.shape
    if dim != fmt.head_dim:
        raise ValueError("query head dimension differs from the page layout")
    _check_float(queries, fmt, "queries")
    device = queries.device
    _check_dense(pool, torch.uint8, device, "pool", 2)
    pages, page_bytes = pool.shape
    if page_bytes != fmt.page_bytes:
        raise ValueError("the pool's pages are not of this format")
    table = _i32(block_table, device)
    if table.dim() != 2 or table.shape[0] != batch:
        raise ValueError("block table must be [batch, max_pages]")
    width = table.shape[1]
    if out is None:
        out = mass if mass is not None else torch.zeros(
            (batch, fmt.num_kv_heads, width * fmt.page_tokens), device=device)
    _check_dense(out, torch.float32, device, "out", 3)
    if mass is not None and mass is not out:
        _check_dense(mass, torch.float32, device, "mass", 3)
        if mass.shape != out.shape:
            raise ValueError("mass and out must have one shape")
    mass_rows, kv_heads, tokens = out.shape
    if kv_heads != fmt.num_kv_heads or (rows is None and mass_rows < batch):
        raise ValueError("attention mass must be [rows, HK, tokens] with a row per sequence")
    lens = _per_row(seq_lens, device, batch, "seq_lens")
    # (the tensors are named so that they live until the launch)
    positions, positions_at = _address(q_pos, device, batch * nq, "q_pos")
    live, live_at = _address(widths, device, batch, "widths")
    known, known_at = _address(counted, device, batch, "counted")
    _distinct(rows, "rows")
    row, row_at = _address(rows, device, batch, "rows")
    queries = queries.contiguous()
    lib, layout = nat.load(), fmt.c_layout
    workspace = _scratch(lib.pkv_attention_mass_workspace_bytes(layout, heads, nq, batch, width),
                         device, "attention mass", workspace)
    _launch(device, "attention mass", lib.pkv_attention_mass, layout, pool.data_ptr(), pages,
            queries.data_ptr(), batch, heads, nq, table.data_ptr(), width, lens.data_ptr(),
            positions_at, live_at, scale, None if mass is None else mass.data_ptr(), known_at,
            row_at, mass_rows, tokens, workspace.data_ptr(), workspace.numel(), out.data_ptr())
    return out


def evict_select(mass, seq_lens, keep, *, max_keep=None, sinks=0, recent=0, rows=None,
                 with_mass=False, new_mass=None):
    """Which tokens of each sequence stay when it is cut down to ``n = min(seq_lens[b],
    keep)``: per layer and KV head the last ``min(recent, n)``, the first ``sinks`` as
    far as there is room, and the heaviest of the others (ties: the lowest index).

    ``mass [R, HK, N]`` or ``[layers, R, HK, N]`` (float32, row ``rows[b]`` or b for
    sequence b); ``keep`` an int, or one per sequence (on the device: with
    ``max_keep``, its bound).  Returns ``(kept [(layers,) B, HK, max_keep] int32``
    ascending, -1 from n on, ``n [B] int32)``; with ``with_mass`` also the kept
    tokens' sums ``[(layers,) R, HK, max_keep]``, in the same order, 0 from n on.
    ``new_mass`` takes them instead (at least ``max_keep`` wide; ``mass`` itself: they
    move in place).
    """
    if mass.dim() not in (3, 4):
        raise ValueError("mass must be [rows, HK, tokens] or [layers, rows, HK, tokens]")
    device = mass.device
    if not mass.is_cuda:
        raise ValueError("mass must be a device tensor")
    _check_dense(mass, torch.float32, device, "mass", mass.dim())
    layers = mass.shape[0] if mass.dim() == 4 else 1
    mass_rows, heads, tokens = mass.shape[-3:]
    lens = _i32(seq_lens, device)
    batch = lens.numel()
    row, row_at = _address(rows, device, batch, "rows")
    if row is None and mass_rows < batch:
        raise ValueError("mass needs a row per sequence")
    if with_mass or new_mass is not None:
        _distinct(rows, "rows")
    if isinstance(keep, int):
        budget_at = None
        if max_keep is None:
            max_keep = keep
        else:
            budget = torch.full((batch,), keep, dtype=torch.int32, device=device)
            budget_at = budget.data_ptr()
    else:
        if max_keep is None:
            if isinstance(keep, torch.Tensor):
                raise ValueError("budgets on the device need max_keep, their bound")
            max_keep = max([int(k) for k in keep], default=0)
        budget, budget_at = _address(keep, device, batch, "keep")
    if _int32(max_keep, "max_keep") < 0:
        raise ValueError("negative budget")
    if sinks < 0 or recent < 0:
        raise ValueError("negative count of protected tokens")
    sinks, recent = min(sinks, max_keep), min(recent, max_keep)
    lead = (layers,) if mass.dim() == 4 else ()
    if new_mass is not None:
        _check_dense(new_mass, torch.float32, device, "new_mass", mass.dim())
        if new_mass.shape[:-1] != mass.shape[:-1] or new_mass.shape[-1] < max_keep:
            raise ValueError("new_mass must be mass's rows of at least max_keep tokens")
    elif with_mass:
        make = torch.empty if row is None and mass_rows == batch else torch.zeros
        new_mass = make(lead + (mass_rows, heads, max_keep), dtype=torch.float32, device=device)
    kept = torch.empty(lead + (batch, heads, max_keep), dtype=torch.int32, device=device)
    new_lens = torch.empty(batch, dtype=torch.int32, device=device)
    sums_at, sums_width = (None, 0) if new_mass is None else (new_mass.data_ptr(),
                                                              new_mass.shape[-1])
    _launch(device, "eviction select", nat.load().pkv_evict_select, mass.data_ptr(), layers,
            mass_rows, heads, tokens, row_at, lens.data_ptr(), batch, budget_at, max_keep, sinks,
            recent, kept.data_ptr(), new_lens.data_ptr(), sums_at, sums_width)
    return (kept, new_lens) if new_mass is None else (kept, new_lens, new_mass)


def evict_pages(fmt: PageFormat, pools, kept, new_lens, src_table, dst_table):
    """Move the ``kept`` tokens of ``evict_select`` from the pages of ``src_table`` to
    positions ``0 .. new_lens[b] - 1`` of those of ``dst_table`` (other pages), K and V,
    bit for bit.

    ``pools``: one pool with ``kept [B, HK, K]``, or a ``[layers, pages, page bytes]``
    tensor or a list of pools with ``kept [layers, B, HK, K]``; one page id addresses
    the same page in every pool.
    """
    device = kept.device
    single = isinstance(pools, torch.Tensor) and pools.dim() == 2
    if isinstance(pools, torch.Tensor):
        _check_dense(pools, torch.uint8, device, "pools", 2 if single else 3)
        layers, shape = (1 if single else pools.shape[0]), pools.shape[-2:]
        step = shape[0] * shape[1]
        addresses = [pools.data_ptr() + i * step for i in range(layers)]
    else:
        for p in pools:
            _check_dense(p, torch.uint8, device, "pools", 2)
        if not pools or any(p.shape != pools[0].shape for p in pools):
            raise ValueError("pools of one call must be of one size")
        layers, shape = len(pools), pools[0].shape
        addresses = [p.data_ptr() for p in pools]
    if shape[1] != fmt.page_bytes:
        raise ValueError("the pools' pages are not of this format")
    _check_dense(kept, torch.int32, device, "kept", 3 if single else 4)
    batch, heads, most = kept.shape[-3:]
    if heads != fmt.num_kv_heads or (not single and kept.shape[0] != layers):
        raise ValueError("kept must be [(layers,) batch, HK, tokens]")
    lens = _per_row(new_lens, device, batch, "new_lens")
    src, dst = _i32(src_table, device), _i32(dst_table, device)
    if src.dim() != 2 or dst.dim() != 2 or src.shape[0] != batch or dst.shape[0] != batch:
        raise ValueError("block tables must be [batch, max_pages]")
    _launch(device, "eviction pages", nat.load().pkv_evict_pages, fmt.c_layout,
            (nat._c_p * layers)(*addresses), layers, shape[0], kept.data_ptr(), lens.data_ptr(),
            batch, most, src.data_ptr(), src.shape[1], dst.data_ptr(), dst.shape[1])


_LOGIT_KINDS = {torch.bfloat16: 0, torch.float16: 1, torch.float32: 2}


def beam_select(logits, scores, count, *, done=None, pad_token=0, workspace=None):
    """The ``count`` best (beam, next token) pairs of every group of beams, by
    ``scores[g, w] + log_softmax(logits[g, w])[v]``, ties to the lowest ``w * V + v``.

    ``logits [G, W, V]`` (float32, bfloat16 or float16; rows may be strided),
    ``scores [G, W]`` float32, ``done [G, W]`` bool: a beam that is done has the one
    candidate ``pad_token`` at its score.  A beam without a finite score and
    log-sum-exp has none; what there are too few of is -inf at the lowest other
    pairs.  Returns ``(scores [G, count] f32, parents int32, tokens int32)`` in
    order, ``parents`` as beam numbers 0..W-1 of the group.
    """
    if logits.dim() != 3 or logits.dtype not in _LOGIT_KINDS or not logits.is_cuda:
        raise ValueError("logits must be a [groups, beams, vocab] f32/f16/bf16 device tensor")
    device = logits.device
    groups, beams, vocab = shape = logits.shape
    group_stride, beam_stride, token_stride = logits.stride()
    if (token_stride != 1 and vocab > 1) or group_stride < 0 or beam_stride < 0:
        logits = logits.contiguous()
        group_stride, beam_stride, _ = logits.stride()
    if scores.shape != shape[:2] or scores.device != device:
        raise ValueError("scores must be [groups, beams] on the logits' device")
    if scores.dtype is not torch.float32 or not scores.is_contiguous():
        scores = scores.to(torch.float32).contiguous()
    done_at = None
    if done is not None:
        if done.shape != shape[:2] or done.dtype is not torch.bool or done.device != device:
            raise ValueError("done must be a [groups, beams] bool tensor on the logits' device")
        done = done.contiguous()
        done_at = done.data_ptr()
    _int32(count, "count")
    _int32(pad_token, "pad_token")
    lib = nat.load()
    workspace = _scratch(lib.pkv_beam_workspace_bytes(groups, beams, vocab, count), device,
                         "beam select", workspace)
    best = torch.empty((groups, count), dtype=torch.float32, device=device)
    parents, tokens = torch.empty((2, groups, count), dtype=torch.int32, device=device).unbind(0)
    _launch(device, "beam select", lib.pkv_beam_select, logits.data_ptr(),
            _LOGIT_KINDS[logits.dtype], groups, beams, vocab, group_stride, beam_stride,
            scores.data_ptr(), done_at, pad_token, count, workspace.data_ptr(), workspace.numel(),
            best.data_ptr(), parents.data_ptr(), tokens.data_ptr())
    return best, parents, tokens


def reorder_rows(state, targets, sources, *, dim=0):
    """Rows of ``state`` along ``dim`` become others' copies, in place and all at once:
    row ``targets[i]`` (distinct) gets what row ``sources[i]`` held before the call.
    Any type; pairs with a row that does not exist are skipped."""
    if not state.is_cuda or not state.is_contiguous():
        raise ValueError("state must be a contiguous device tensor")
    if not 0 <= dim < state.dim():
        raise ValueError("no such dimension")
    device = state.device
    _distinct(targets, "targets")
    to, source = _i32(targets, device), _i32(sources, device)
    count = to.numel()
    if source.numel() != count:
        raise ValueError("reordering needs a source per target")
    shape = state.shape
    outer, num_rows = math.prod(shape[:dim]), _int32(shape[dim], "the number of rows")
    row_bytes = math.prod(shape[dim + 1:]) * state.element_size()
    _launch(device, "reorder", nat.load().pkv_reorder_rows, state.data_ptr(), outer, num_rows,
            row_bytes, to.data_ptr(), source.data_ptr(), count)
    return state


# ---- a serving step ------------------------------------------------------------------


def rope_append(fmt: PageFormat, pool, qkv, block_table, start_pos, inv_freq, heads, *, row_starts=None,
                widths=None, positions=None, axes=None, with_kv=False, out=None):
    """Rotate the q and k heads of a fused projection and store k and v into the
    sequences' pages, in one pass; returns the rotated q.

    ``qkv`` holds ``heads`` query heads, then k and v of the format's KV heads, in rows of
    ``(heads + 2 * HK) * D`` elements: packed ``[T, width]`` with ``row_starts [B + 1]`` (sequence
    b has rows ``row_starts[b]`` to ``row_starts[b + 1] - 1``), or padded ``[B, N, width]`` with
    ``widths [B]`` (default: N).  Row i of sequence b is appended at ``start_pos[b] + i``.

    The first ``2 * len(inv_freq)`` elements of a head are rotated (rotate-half pairs), by the
    cache position or by ``positions``, ``[T]`` (padded ``[B, N]``); positions on several axes,
    ``[A, T]`` (``[A, B, N]``), go with ``axes [len(inv_freq)]``, the axis of each frequency.  Angles
    are in 64 bits.  The pages equal ``append_quantize``'s of the k and v that come out, bit
    for bit.

    Returns q ``[T, heads, D]`` (padded ``[B, heads, N, D]``); ``with_kv`` also k and v, with HK
    heads.  ``out``: a tensor, or with ``with_kv`` three, that take them; rows of no
    sequence are left as they are there.
    """
    if not isinstance(qkv, torch.Tensor) or qkv.dim() != (3 if row_starts is None else 2):
        raise ValueError("qkv must be packed [T, width] with row_starts, or padded [B, N, width]")
    _check_float(qkv, fmt, "qkv")
    device = qkv.device
    _check_dense(pool, torch.uint8, device, "pool", 2)
    if pool.shape[1] != fmt.page_bytes:
        raise ValueError("the pool's pages are not of this format")
    kv_heads, dim = fmt.num_kv_heads, fmt.head_dim
    *lead, width = qkv.shape
    if heads < 1 or width != (heads + 2 * kv_heads) * dim:
        raise ValueError("qkv width is not (heads + 2 * kv_heads) * head_dim")
    qkv, step = _projection_rows(qkv)
    starts = _i32(start_pos, device)
    batch = starts.numel()
    # (the tensors are named so that they live until the launch)
    if row_starts is None:
        if widths is not None:
            widths, widths_at = _address(widths, device, batch, "widths")
        else:
            widths_at = None
        if lead[0] != batch:
            raise ValueError("start_pos must hold a value per sequence")
        tokens, first_at = lead[1], None
        rows = batch * tokens
    else:
        if widths is not None:
            raise ValueError("packed rows take no widths")
        rows, tokens, widths_at = lead[0], 0, None
        first, first_at = _address(row_starts, device, batch + 1, "row_starts")
    table = _i32(block_table, device)
    if table.dim() != 2 or table.shape[0] != batch:
        raise ValueError("block table must be [batch, max_pages]")
    _check_dense(inv_freq, torch.float32, device, "inv_freq", 1)
    half = inv_freq.shape[0]
    num_axes, positions_at, axis_at = 1, None, None
    if positions is not None:
        places = _i32(positions, device)
        if axes is not None and places.dim() == len(lead) + 1:
            num_axes = places.shape[0]
        if [*places.shape] != [num_axes] * (axes is not None) + lead:
            raise ValueError("positions must be one per row, or with axes one per axis and row")
        positions_at = places.data_ptr()
    if axes is not None:
        if positions is None:
            raise ValueError("axes need positions")
        axis, axis_at = _address(axes, device, half, "axes")
    shapes = [(rows, n, dim) if row_starts is not None else (batch, n, tokens, dim)
              for n in ((heads, kv_heads, kv_heads) if with_kv else (heads,))]
    if out is None:
        outs = [torch.empty(shape, dtype=qkv.dtype, device=device) for shape in shapes]
    else:
        outs = list(out) if with_kv else [out]
        if len(outs) != len(shapes):
            raise ValueError("out must hold q, k and v")
        for t, shape in zip(outs, shapes):
            if not _dense(t, qkv.dtype, device, len(shape)) or t.shape != shape:
                raise ValueError(f"out must be contiguous {shape} tensors of qkv's dtype and device")
    addresses = [t.data_ptr() for t in outs] if with_kv else (outs[0].data_ptr(), None, None)
    _launch(device, "rotation and append", nat.load().pkv_rope_append, fmt.c_layout, pool.data_ptr(),
            pool.shape[0], qkv.data_ptr(), step, rows, heads, batch, tokens, first_at, widths_at,
            starts.data_ptr(), positions_at, num_axes, inv_freq.data_ptr(), half, axis_at,
            table.data_ptr(), table.shape[1], *addresses)
    return tuple(outs) if with_kv else outs[0]


def _projection_rows(qkv):
    """A projection ``[rows, width]`` or ``[B, N, width]`` as the kernels read it, its rows one
    after the other (a copy where they are not): ``(tensor, elements between rows)``.  A
    dimension of one element has any stride, which says nothing."""
    *lead, width = qkv.shape
    steps = [(n, step) for n, step in zip(lead, qkv.stride()) if n != 1]
    step = steps[-1][1] if steps else width
    if qkv.stride(-1) != 1 or step < width or (len(steps) == 2 and steps[0][1] != steps[1][0] * step):
        return qkv.clone(memory_format=torch.contiguous_format), width
    return qkv, step


def rope_axes(sections, device="cuda", *, interleaved=False):
    """The axis of each frequency for ``rope_append``: runs of ``sections[a]`` frequencies for axis
    a, or, interleaved, the axes in turn, each as long as it has any of its ``sections[a]``
    left."""
    counts = [int(n) for n in sections]
    if not counts or any(n < 0 for n in counts):
        raise ValueError("sections must be counts of frequencies")
    if interleaved:
        order = [a for i in range(max(counts)) for a, n in enumerate(counts) if i < n]
    else:
        order = [a for a, n in enumerate(counts) for _ in range(n)]
    return torch.tensor(order, dtype=torch.int32, device=device)


def _packed_rows(t, rows, heads, dim):
    """Packed heads ``[T, heads, D]`` as the kernels read them: heads side by side, rows any
    multiple of 16 bytes apart (a copy where they are not).  ``(tensor, address, stride of
    rows)``."""
    step, head_step, one = t.stride()
    at = t.data_ptr()
    if rows > 0 and (one != 1 or (head_step != dim and heads > 1) or step < heads * dim or step % 8
                     or step > 1 << 23 or at % 16):
        t = t.clone(memory_format=torch.contiguous_format)
        at, step = t.data_ptr(), heads * dim
    return t, at, (step if rows > 1 else heads * dim)


def prompt_attention(q, k, v, row_starts, *, scale, out=None):
    """Causal attention within every sequence of packed rows.

    ``q [T, H, D]``, ``k`` and ``v [T, HK, D]`` (bfloat16 or float16; views of a fused projection
    are read where they lie); sequence b is rows ``row_starts[b]`` to ``row_starts[b + 1] - 1``
    (``row_starts [B + 1]``, rising).  Returns ``[T, H, D]``; rows of no sequence are left as they
    are in ``out``.  Head dims up to 256; ones that are no multiple of 8 are padded by a copy.
    Weights are rounded to the inputs' type, where ``paged_attention`` over bfloat16 pages keeps
    them as the sum of two.
    """
    for t in (q, k, v):
        if not isinstance(t, torch.Tensor) or t.dim() != 3 or t.dtype not in FLOAT_KINDS or not t.is_cuda:
            raise ValueError("q, k and v must be [T, heads, D] f16/bf16 device tensors")
    rows, heads, dim = q.shape
    device, dtype = q.device, q.dtype
    key_rows, kv_heads, key_dim = k.shape
    if k.shape != v.shape or key_rows != rows or key_dim != dim:
        raise ValueError("k and v must be [T, HK, D] of q's rows and head dimension")
    if k.dtype is not dtype or v.dtype is not dtype or k.device != device or v.device != device:
        raise ValueError("q, k and v must be of one dtype and device")
    starts = _i32(row_starts, device)
    if starts.dim() != 1 or starts.numel() < 1:
        raise ValueError("row_starts must be [batch + 1]")
    if out is not None and (not _dense(out, dtype, device, 3) or out.shape != q.shape):
        raise ValueError("out must be a contiguous tensor of q's shape, dtype and device")
    result, width = out, dim
    if dim % 8:
        width = dim + 8 - dim % 8
        q, k, v = (torch.nn.functional.pad(t, (0, width - dim)) for t in (q, k, v))
        out = None
    if out is None or out.data_ptr() % 16:
        out = torch.empty((rows, heads, width), dtype=dtype, device=device)
        if result is not None:
            out[..., :dim] = result
    # (the tensors are named so that they live until the launch)
    q, q_at, q_step = _packed_rows(q, rows, heads, width)
    k, k_at, k_step = _packed_rows(k, rows, kv_heads, width)
    v, v_at, v_step = _packed_rows(v, rows, kv_heads, width)
    _launch(device, "prompt attention", nat.load().pkv_prompt_attention, q_at, q_step, k_at, k_step, v_at, v_step,
            FLOAT_KINDS[dtype], rows, starts.numel() - 1, starts.data_ptr(), heads, kv_heads, width, scale,
            out.data_ptr())
    if result is None:
        return out if width == dim else out[..., :dim].contiguous()
    if result is not out:
        result.copy_(out[..., :dim])
    return result


def shared_workspace_bytes(fmt: PageFormat, heads, queries, members, groups):
    """Workspace of ``shared_prefix_attention`` for as many members and groups, whatever their
    lengths."""
    need = int(nat.load().pkv_shared_attention_workspace_bytes(fmt.c_layout, heads, queries, members, groups))
    if need < 0:
        nat.check(-need, "shared attention")
    return need


def shared_prefix_attention(fmt: PageFormat, pool, queries, block_table, seq_lens, members, group_starts,
                            prefix_lens, *, scale, q_pos=None, widths=None, workspace=None, out=None):
    """Attention of ``queries [B, H, Q, D]`` over the paged cache, where the sequences of a
    group hold the same first tokens: these are gone through once for the group.

    Group g is sequences ``members[group_starts[g]:group_starts[g + 1]]`` (distinct) and shares
    its first ``prefix_lens[g]`` tokens -- pages that ``fork`` shares, or equal copies.  The other
    operands and the result are ``paged_attention``'s (at most 32 query rows per KV head, 16
    beyond head dim 128, 1024 sequences); rows of sequences that no group names are
    left as they are in ``out``, or zero.
    """
    if queries.dim() != 4:
        raise ValueError("queries must be [B, H, Q, D]")
    batch, heads, nq, dim = queries.shape
    if dim != fmt.head_dim:
        raise ValueError("query head dimension differs from the page layout")
    _check_float(queries, fmt, "queries")
    device = queries.device
    _check_dense(pool, torch.uint8, device, "pool", 2)
    pages, page_bytes = pool.shape
    if page_bytes != fmt.page_bytes:
        raise ValueError("the pool's pages are not of this format")
    table = _i32(block_table, device)
    if table.dim() != 2 or table.shape[0] != batch:
        raise ValueError("block table must be [batch, max_pages]")
    lens = _per_row(seq_lens, device, batch, "seq_lens")
    # (the tensors are named so that they live until the launch)
    positions, positions_at = _address(q_pos, device, batch * nq, "q_pos")
    live, live_at = _address(widths, device, batch, "widths")
    _distinct(members, "members")
    member = _i32(members, device)
    count = member.numel()
    starts, prefix = _i32(group_starts, device), _i32(prefix_lens, device)
    groups = prefix.numel()
    if starts.numel() != groups + 1:
        raise ValueError("group_starts must hold a value per group and the end")
    queries = queries.contiguous()
    fresh = out is None
    if fresh:
        out = (torch.empty if count and groups else torch.zeros)(queries.shape, dtype=queries.dtype, device=device)
    elif not _dense(out, queries.dtype, device, 4) or out.shape != queries.shape:
        raise ValueError("out must be a contiguous tensor of the queries' shape, dtype and device")
    lib, layout = nat.load(), fmt.c_layout
    workspace = _scratch(shared_workspace_bytes(fmt, heads, nq, count, groups), device, "shared attention", workspace)
    _launch(device, "shared attention", lib.pkv_shared_attention, layout, pool.data_ptr(), pages, queries.data_ptr(),
            batch, heads, nq, table.data_ptr(), table.shape[1], lens.data_ptr(), positions_at, live_at, groups,
            member.data_ptr(), count, starts.data_ptr(), prefix.data_ptr(), scale, workspace.data_ptr(),
            workspace.numel(), out.data_ptr(), fresh)
    return out
