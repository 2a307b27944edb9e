"""A serving step on the paged cache, from the fused projection to the attention output:
rotation and append in one pass, attention over packed prompts, and attention of a
batch whose sequences share a long prefix.

A case is a plain dict.  ``kind`` says which operator a pass runs:

* ``rope``   -- rows of a fused q|k|v projection, packed over sequences: q and k are
  rotated at their positions (on one axis, or on three for image and video tokens),
  k and v are stored into the sequences' pages, q (and k and v) come out.
* ``prompt`` -- causal attention within every sequence of packed rows, grouped heads.
* ``shared`` -- decode or verify queries over pages, where the sequences of a group hold
  the same first pages.

Where ``own`` is false a pass computes the operator in elementary torch operations
over the same tensors; where it is true it makes this package's calls.  Lengths are
spread by a fixed rule, so a case's sizes do not depend on the seed.
"""

import math
import os
import sys

import numpy as np
import torch

_PACKAGE = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "mlx-one_amd")
if _PACKAGE not in sys.path:
    sys.path.insert(0, _PACKAGE)

own = False

_DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16}


def listed():
    return [
        # one step of a small model: launches and host calls are all there is
        _rope("rope_bf16_small", batch=4, heads=8, kv_heads=2, dim=64, bits=16, lo=1, hi=1, cached=400),
        # a serving batch's next tokens, 1K..8K tokens in
        _rope("rope_int8_decode", batch=64, lo=1, hi=1, cached=8000),
        # prompts of a chat batch, whose attention wants k and v as well
        _rope("rope_int8_prompts", batch=12, lo=150, hi=3900, cached=0, with_kv=True),
        # image tokens (time, height, width) on 4-bit pages, behind some text
        _rope("rope_int4_axes", batch=8, heads=16, kv_heads=2, bits=4, group=32, page=32, dtype="f16", lo=900,
              hi=1700, cached=37, axes=3),
        # a few short prompts of a small model
        _prompt("prompt_f16_small", batch=3, heads=8, kv_heads=2, dim=64, dtype="f16", lo=17, hi=200),
        # a serving batch of prompts of different lengths
        _prompt("prompt_bf16_mixed", batch=16, lo=100, hi=2000),
        # one long document
        _prompt("prompt_bf16_long", batch=1, lo=16000, hi=16000),
        # wide heads
        _prompt("prompt_bf16_dim256", batch=4, heads=16, kv_heads=4, dim=256, lo=700, hi=2100),
        # four short chats behind one instruction
        _shared("shared_bf16_small", batch=4, heads=8, kv_heads=2, dim=64, bits=16, prefix=256, lo=10, hi=60),
        # a serving batch behind one long system prompt
        _shared("shared_int8_b32", batch=32, prefix=4096, lo=64, hi=2000),
        # several answers to each of four long documents, eight heads per KV head
        _shared("shared_int4_documents", batch=32, groups=4, heads=32, kv_heads=4, page=32, bits=4, prefix=24000,
                lo=20, hi=300),
        # verify steps of five tokens, four instructions
        _shared("shared_int8_verify", batch=16, groups=4, queries=5, prefix=2000, lo=5, hi=700),
    ]


def _case(kind, kw):
    case = dict(kind=kind, batch=1, heads=32, kv_heads=8, dim=128, page=16, bits=8, group=64, dtype="bf16", lo=1, hi=1)
    case.update(kw)
    return case


def _rope(name, **kw):
    return dict(name=name, **_case("rope", dict(dict(axes=1, rotated=1.0, with_kv=False), **kw)))


def _prompt(name, **kw):
    case = dict(name=name, **_case("prompt", kw))
    for key in ("page", "bits", "group"):
        del case[key]
    return case


def _shared(name, **kw):
    return dict(name=name, **_case("shared", dict(dict(groups=1, queries=1), **kw)))


def _spread(rng, lo, hi):
    """A size of lo..hi, spread over its logarithm."""
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    most = max(_cost(c) for c in listed())
    while True:
        kind = rng.choice(["rope", "prompt", "shared"])
        dim = rng.choice([64, 128, 128, 128, 96, 80, 256])
        kv_heads = rng.choice([1, 2, 4, 8, 8])
        heads = kv_heads * rng.choice([1, 2, 4, 4, 7, 8])
        case = dict(kind=kind, batch=_spread(rng, 1, 64), heads=heads, kv_heads=kv_heads, dim=dim,
                    dtype=rng.choice(["bf16", "bf16", "f16"]))
        if kind != "prompt":
            case.update(bits=rng.choice([8, 8, 4, 4, 16]), page=rng.choice([16, 16, 32, 64, 128]),
                        group=rng.choice([g for g in (32, 64, 128) if g <= max(64, dim // 2)]))
        if kind == "rope":
            lo = rng.choice([1, 1, _spread(rng, 2, 4000)])
            case.update(lo=lo, hi=lo if lo == 1 else min(8000, lo + _spread(rng, 1, 2 * lo)),
                        cached=rng.choice([0, _spread(rng, 1, 20000)]), axes=rng.choice([1, 1, 3]),
                        rotated=rng.choice([1.0, 1.0, 0.5]), with_kv=rng.choice([False, True]))
        elif kind == "prompt":
            lo = _spread(rng, 1, 12000)
            case.update(lo=lo, hi=min(16000, lo + _spread(rng, 1, 2 * lo)))
        else:
            lo = _spread(rng, 1, 2000)
            case.update(groups=rng.randint(1, max(1, case["batch"] // 2)), prefix=_spread(rng, 17, 32000), lo=lo,
                        hi=lo + _spread(rng, 1, 2 * lo), queries=rng.choice([1, 1, 1, rng.randint(2, 8)]))
            if case["queries"] * heads // kv_heads > 32:
                continue
        if _cost(case) <= 0.8 * most and _held(case) <= 1.5e9 and _plain_bytes(case) <= 3e10:
            return case


# ---- sizes -------------------------------------------------------------------------


def _lengths(case):
    """New tokens (shared: tokens behind the prefix) per sequence."""
    n, lo, hi = case["batch"], case["lo"], case["hi"]
    return [lo + int((hi - lo) * ((i + 1) * 0.6180339887498949 % 1.0)) if n > 1 else hi for i in range(n)]


def _cached(case):
    """Tokens in the cache before a rope pass."""
    most = case["cached"]
    return [most // 8 + int((most - most // 8) * ((i + 1) * 0.7548776662466927 % 1.0)) for i in range(case["batch"])]


def _prefixes(case):
    """Shared tokens per group: whole pages."""
    page, most = case["page"], case["prefix"]
    return [(most - int(0.25 * most * (g * 0.6180339887498949 % 1.0))) // page * page for g in range(case["groups"])]


def _group_of(case, b):
    return b % case["groups"]


def _geometry(case):
    """The page layout's sizes: stored dim, groups, payload and metadata bytes of a head block's side."""
    bits, group, dim = case["bits"], case["group"], case["dim"]
    need = dim if bits == 16 else -(-dim // group) * group
    dp = 64 if need <= 64 else 128 if need <= 128 else 256
    groups = 0 if bits == 16 else dp // group
    return dp, groups, case["page"] * dp * bits // 8, case["page"] * groups * 4


def _side_bytes(case):
    """Bytes of one token's K (or V) in one head."""
    if case["bits"] == 16:
        return 2 * case["dim"]
    groups = -(-case["dim"] // case["group"])
    return groups * case["group"] * case["bits"] // 8 + 4 * groups


def _rotary(case):
    """Rotated elements of a head."""
    return int(case["dim"] * case["rotated"]) // 16 * 16


def work(case):
    h, hk, d = case["heads"], case["kv_heads"], case["dim"]
    lengths = _lengths(case)
    tokens = sum(lengths)
    if case["kind"] == "rope":
        elements = (2 * h + 2 * hk + (2 * hk if case["with_kv"] else 0)) * d
        return {"bytes": tokens * (2 * elements + 2 * hk * _side_bytes(case) + 4 * case["axes"]),
                "flops": 3 * tokens * (h + hk) * _rotary(case)}
    if case["kind"] == "prompt":
        return {"bytes": 4 * tokens * (h + hk) * d, "flops": 2 * d * h * sum(n * (n + 1) for n in lengths)}
    q, prefixes = case["queries"], _prefixes(case)
    pairs = sum(q * (prefixes[_group_of(case, b)] + n) - q * (q - 1) // 2 for b, n in enumerate(lengths))
    return {"bytes": (sum(prefixes) + tokens) * hk * 2 * _side_bytes(case) + 4 * case["batch"] * h * q * d,
            "flops": 4 * d * h * pairs}


def _cost(case):
    w = work(case)
    return max(w["bytes"], w["flops"] / 200)


def _pages(case):
    """Pages that a state's sequences hold."""
    page = case["page"]
    if case["kind"] == "rope":
        return sum(-(-(c + n) // page) for c, n in zip(_cached(case), _lengths(case)))
    return sum(p // page for p in _prefixes(case)) + sum(-(-n // page) for n in _lengths(case))


def _held(case):
    """Bytes that a state holds, roughly."""
    if case["kind"] == "prompt":
        return work(case)["bytes"]
    _, _, payload, meta = _geometry(case)
    return _pages(case) * case["kv_heads"] * 2 * (payload + meta) + work(case)["bytes"]


def _plain_bytes(case):
    """Bytes of the largest tensor of a plain pass, roughly."""
    if case["kind"] == "rope":
        return 40 * work(case)["bytes"]
    if case["kind"] == "prompt":
        return 4 * case["batch"] * case["heads"] * max(_lengths(case)) ** 2
    longest = max(_prefixes(case)) + max(_lengths(case)) + case["page"]
    return 4 * case["batch"] * longest * max(case["heads"] * case["queries"], case["kv_heads"] * 256)


# ---- inputs ------------------------------------------------------------------------


def _generator(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(int(seed) * 6007 + 41)
    return g


def _ints(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def _starts(lengths):
    return _ints([0] + np.cumsum(lengths).tolist())


def _quantized(case, x):
    """Codes [..., dp] u8 and (scale, bias) words [..., groups] of rows x [..., dp]."""
    levels = torch.tensor(float(2 ** case["bits"] - 1), device=x.device)  # (a tensor: divided by, not multiplied)
    x = x.float().unflatten(-1, (-1, case["group"]))
    low = x.amin(-1, keepdim=True).half()
    step = ((x.amax(-1, keepdim=True) - low.float()) / levels).clamp_min(1e-6).half()
    codes = ((x - low.float()) / step.float()).round().clamp(0, 2 ** case["bits"] - 1).to(torch.uint8).flatten(-2)
    words = torch.stack((step, low), -1).squeeze(-2).contiguous().view(torch.int32).squeeze(-1)
    return codes, words


def _random_pool(case, gen, pages):
    """A pool of `pages` pages, [pages, page bytes] u8: K and V rows N(0, 1) with a few larger
    head-dim channels, as quantized codes (or floats) and their (scale, bias) words.  Elements are
    made in the order that the pages store them in: they are alike in every place."""
    dp, groups, payload, meta = _geometry(case)
    shape = (pages, case["kv_heads"])
    if case["bits"] == 16:
        # a lane's elements: K 8 dims of a token, V 4 tokens of a dim; dims past the head's hold zeros
        k = torch.randn(shape + (case["page"] // 16, dp // 32, 4, 16, 8), generator=gen, device="cuda")
        v = torch.randn(shape + (case["page"] // 16, dp // 32, 4, 16, 2, 4), generator=gen, device="cuda")
        d = torch.arange(dp, device="cuda")
        k *= (d < case["dim"]).view(dp // 32, 4, 1, 8)
        v *= (d < case["dim"]).view(dp // 32, 2, 16).permute(0, 2, 1).reshape(dp // 32, 1, 16, 2, 1)
        both = torch.cat((k.flatten(2), v.flatten(2)), -1).to(_DTYPES[case["dtype"]])
        return both.view(torch.uint8).flatten(1)
    codes = torch.randint(0, 256, shape + (2 * payload,), generator=gen, device="cuda", dtype=torch.uint8)
    # a group of N(0, 1) values spans about five, a few groups more
    span = 4 + 2 * torch.rand(shape + (2 * meta // 4,), generator=gen, device="cuda")
    span = span * torch.where(torch.rand(span.shape, generator=gen, device="cuda") < 0.05, 2.0, 1.0)
    words = torch.stack(((span / (2 ** case["bits"] - 1)).half(), (-span / 2).half()), -1)
    return torch.cat((codes, words.view(torch.uint8).flatten(2)), -1).flatten(1)


def _inverse_frequencies(case):
    half = _rotary(case) // 2
    return (500000.0 ** (-torch.arange(half, dtype=torch.float64, device="cuda") / half)).float()


def _axis_map(case):
    """The axis of every frequency: runs of a quarter, and the rest in halves."""
    half = _rotary(case) // 2
    first = half // 4
    second = first + (half - first) // 2
    i = torch.arange(half, device="cuda")
    return ((i >= first).int() + (i >= second).int()).to(torch.int32)


def prepare(case, seed):
    gen = _generator(seed)
    s = dict(case)
    dtype, lengths = _DTYPES[case["dtype"]], _lengths(case)
    h, hk, d, batch = case["heads"], case["kv_heads"], case["dim"], case["batch"]

    def rows(*shape):
        return torch.randn(shape, generator=gen, device="cuda").to(dtype)

    if case["kind"] == "prompt":
        total = sum(lengths)
        s["q"], s["k"], s["v"] = rows(total, h, d), rows(total, hk, d), rows(total, hk, d)
        s["starts"] = _starts(lengths)
        return s
    page = case["page"]
    ids = np.random.default_rng(seed).permutation(_pages(case)).astype(np.int32)
    s["pool"] = _random_pool(case, gen, len(ids))
    at = 0
    if case["kind"] == "rope":
        cached, total = _cached(case), sum(lengths)
        counts = [-(-(c + n) // page) for c, n in zip(cached, lengths)]
        table = np.full((batch, max(counts)), -1, np.int32)
        for b, n in enumerate(counts):
            table[b, :n] = ids[at:at + n]
            at += n
        gain = torch.ones((h + 2 * hk, d), device="cuda")
        gain[:, torch.randperm(d, generator=gen, device="cuda")[:2]] = 3.0
        s["qkv"] = (torch.randn((total, (h + 2 * hk) * d), generator=gen, device="cuda") * gain.flatten()).to(dtype)
        s["starts"], s["cached_lens"] = _starts(lengths), _ints(cached)
        s["inv_freq"] = _inverse_frequencies(case)
        if case["axes"] > 1:
            s["axis"] = _axis_map(case)
            # image patches, row by row, behind the cached text
            i = torch.arange(total, device="cuda") - torch.repeat_interleave(s["starts"][:-1], _ints(lengths))
            first = torch.repeat_interleave(s["cached_lens"], _ints(lengths))
            side = max(1, int(math.isqrt(max(lengths))))
            turn = int(torch.randint(0, 50, (1,), generator=gen, device="cuda"))
            s["positions"] = torch.stack((first + turn, first + i // side, first + i % side)).to(torch.int32)
    else:
        prefixes = _prefixes(case)
        held = []
        for p in prefixes:
            held.append(ids[at:at + p // page])
            at += p // page
        counts = [-(-n // page) for n in lengths]
        width = max(prefixes[_group_of(case, b)] // page + n for b, n in enumerate(counts))
        table = np.full((batch, width), -1, np.int32)
        for b, n in enumerate(counts):
            first = held[_group_of(case, b)]
            table[b, :len(first)] = first
            table[b, len(first):len(first) + n] = ids[at:at + n]
            at += n
        s["lens"] = _ints([prefixes[_group_of(case, b)] + n for b, n in enumerate(lengths)])
        members = [[b for b in range(batch) if _group_of(case, b) == g] for g in range(case["groups"])]
        s["members"] = _ints([b for m in members for b in m])
        s["group_starts"] = _starts([len(m) for m in members])
        s["prefix_lens"] = _ints(prefixes)
        s["q"] = rows(batch, h, case["queries"], d)
    s["table"] = torch.from_numpy(table).cuda()
    return s


# ---- one pass ------------------------------------------------------------------------


def run(state):
    return (_OWN if own else _PLAIN)[state["kind"]](state)


def _format(s):
    """The layer's page format, made once and kept with the pool."""
    from pkv import ops

    if "fmt" not in s:
        s["fmt"] = ops.PageFormat(s["kv_heads"], s["dim"], s["page"], s["bits"], s["group"], _DTYPES[s["dtype"]])
    return s["fmt"]


def _own_rope(s):
    from pkv import ops

    out = ops.rope_append(_format(s), s["pool"], s["qkv"], s["table"], s["cached_lens"], s["inv_freq"], s["heads"],
                          row_starts=s["starts"], positions=s.get("positions"), axes=s.get("axis"),
                          with_kv=s["with_kv"])
    if s["with_kv"]:
        return {"q": out[0], "k": out[1], "v": out[2], "pages": _page_values(s)}
    return {"q": out, "pages": _page_values(s)}


def _own_prompt(s):
    from pkv import ops

    return ops.prompt_attention(s["q"], s["k"], s["v"], s["starts"], scale=s["dim"] ** -0.5)


def _own_shared(s):
    from pkv import ops

    return ops.shared_prefix_attention(_format(s), s["pool"], s["q"], s["table"], s["lens"], s["members"],
                                       s["group_starts"], s["prefix_lens"], scale=s["dim"] ** -0.5)


_OWN = {"rope": _own_rope, "prompt": _own_prompt, "shared": _own_shared}


def _page_values(s):
    """The pages a pass has written, whole: float pages as their values; codes and (scale, bias)
    words as they are stored.  They are whole numbers that follow from k and v, rounded to the
    activation type, by IEEE operations alone, so two computations of them agree in every bit."""
    return s["pool"].view(_DTYPES[s["dtype"]]) if s["bits"] == 16 else s["pool"]


# Where a token's elements sit in a head block: K tiles, V tiles (16 tokens each), then for quantized
# pages the K and V metadata words.  A tile is chunks of 64 lanes of `cs` bytes; K's lane 16*jj + t holds
# dims 32*kb + 8*jj + e of token t, V's lane 16*jj + c holds tokens 4*jj + r of dims 16*n + c.


def _chunk_bytes(case):
    return min(16, _geometry(case)[0] * case["bits"] // 32)


def _lane_place(case, lane, byte):
    cs = _chunk_bytes(case)
    return byte // cs * (64 * cs) + lane * cs + byte % cs


def _token_places(case, slot):
    """Byte offsets in a head block of the K and V elements of the token in `slot` [T]: [T, dp] each
    (4-bit: of the pairs of codes that share a byte, [T, dp / 2])."""
    dp, _, payload, _ = _geometry(case)
    bits = case["bits"]
    tile, t = (slot // 16 * (dp * bits * 2))[:, None], (slot % 16)[:, None]
    x = torch.arange(dp // 2 if bits == 4 else dp, device=slot.device)
    if bits == 4:
        # K: dword kb of lane jj, byte y: codes (0, 2), (4, 6), (1, 3), (5, 7); V: dims 32*m + c and + 16
        kb, jj, y = x // 16, x // 4 % 4, x % 4
        k = _lane_place(case, t + 16 * jj, 4 * kb + y)
        order = torch.tensor([0, 2, 1, 3], device=slot.device)
        v = _lane_place(case, x % 16 + t // 4 * 16, 4 * (x // 16) + order[t % 4])
    else:
        size = bits // 8
        k = _lane_place(case, t + 16 * (x % 32 // 8), size * (8 * (x // 32) + x % 8))
        v = _lane_place(case, x % 16 + t // 4 * 16, size * (4 * (x // 16) + t % 4))
    return tile + k, payload + tile + v


def _packed4(codes):
    """4-bit codes [..., dp] as the bytes of _token_places: (K's, V's)."""
    k = codes.unflatten(-1, (-1, 4, 8))
    k = k[..., [0, 4, 1, 5]] | (k[..., [2, 6, 3, 7]] << 4)
    v = codes.unflatten(-1, (-1, 2, 16))
    return k.flatten(-3), (v[..., 0, :] | (v[..., 1, :] << 4)).flatten(-2)


def _plain_rope(s):
    h, hk, d, half = s["heads"], s["kv_heads"], s["dim"], _rotary(s) // 2
    dtype, total = _DTYPES[s["dtype"]], s["qkv"].shape[0]
    rows = torch.arange(total, device="cuda")
    b = torch.searchsorted(s["starts"][1:].long().contiguous(), rows, right=True)
    position = rows - s["starts"].long()[b] + s["cached_lens"].long()[b]
    # angles in 64 bits: those of far positions keep no digit behind the point in 32
    where = s["positions"].long()[s["axis"].long()].t() if "positions" in s else position[:, None]
    angle = where.double() * s["inv_freq"].double()
    cos, sin = (f(angle).float()[:, None] for f in (torch.cos, torch.sin))
    x = s["qkv"].view(total, h + 2 * hk, d)
    turned = x[:, :h + hk].float()
    first, second = turned[..., :half].clone(), turned[..., half:2 * half].clone()
    turned[..., :half] = first * cos - second * sin
    turned[..., half:2 * half] = second * cos + first * sin
    turned = turned.to(dtype)
    q, k, v = turned[:, :h].contiguous(), turned[:, h:].contiguous(), x[:, h + hk:].contiguous()
    dp, groups, payload, meta = _geometry(s)
    page = s["table"].long()[b, position // s["page"]]
    slot = position % s["page"]
    head = 2 * (payload + meta)
    base = (page[:, None] * hk + torch.arange(hk, device="cuda"))[..., None] * head       # [T, HK, 1]
    sides = [torch.nn.functional.pad(y, (0, dp - d)) for y in (k, v)]
    if s["bits"] == 16:
        flat = s["pool"].view(-1).view(torch.int16)
        for y, place in zip(sides, _token_places(s, slot)):
            flat[(base + place[:, None]) // 2] = y.view(torch.int16)
    else:
        for i, (y, place) in enumerate(zip(sides, _token_places(s, slot))):
            codes, words = _quantized(s, y)
            if s["bits"] == 4:
                codes = _packed4(codes)[i]
            s["pool"].view(-1)[base + place[:, None]] = codes
            at = (2 * payload + i * meta + 4 * slot * groups)[:, None] + 4 * torch.arange(groups, device="cuda")
            s["pool"].view(-1).view(torch.int32)[(base + at[:, None]) // 4] = words
    out = {"q": q, "pages": _page_values(s)}
    return dict(out, k=k, v=v) if s["with_kv"] else out


def _plain_prompt(s):
    h, hk, d, batch = s["heads"], s["kv_heads"], s["dim"], s["batch"]
    starts = s["starts"].long()
    lengths = starts[1:] - starts[:-1]
    longest = max(_lengths(s))                                                       # (known to the program)
    at = torch.arange(longest, device="cuda")
    there = at < lengths[:, None]                                                    # [B, N]
    rows = (starts[:-1, None] + at).clamp_max(s["q"].shape[0] - 1)
    q, k, v = (s[name][rows].float().transpose(1, 2).contiguous() for name in "qkv")  # [B, heads, N, D]
    q = q.view(batch * hk, -1, d)                                                    # the heads of a KV head together
    scores = q @ (k.flatten(0, 1) * d ** -0.5).transpose(1, 2).contiguous()
    scores = scores.view(batch, hk, -1, longest, longest)
    scores.masked_fill_((at > at[:, None]) | ~there[:, None, None, None], -math.inf)
    scores -= scores.amax(-1, keepdim=True).clamp_min(-1e30)
    scores.exp_()
    scores /= scores.sum(-1, keepdim=True).clamp_min(1e-30)
    out = scores.view(batch * hk, -1, longest) @ v.flatten(0, 1)
    out = out.view(batch, h, longest, d).transpose(1, 2)
    return out[there].to(_DTYPES[s["dtype"]])


_K4 = [0, 4, 1, 5, 2, 6, 3, 7]  # the nibble of a K word's element e
_V4 = [0, 2, 1, 3]              # the byte of a V word's token r


def _elements(case, payload):
    """Lane bytes [..., cs] as elements in the lane's order: int16, u8, or a nibble per u8."""
    if case["bits"] == 16:
        return payload.view(torch.int16)
    return payload if case["bits"] == 8 else torch.stack((payload & 15, payload >> 4), -1).flatten(-2)


def _tokens(case, payload, values):
    """K or V payload bytes [..., payload] as elements [..., page, dp]."""
    cs = _chunk_bytes(case)
    lead, n = payload.shape[:-1], payload.dim() - 1
    chunks = _geometry(case)[0] * case["bits"] // 32 // cs
    x = _elements(case, payload.reshape(*lead, -1, chunks, 4, 16, cs))
    if values:
        if case["bits"] == 4:                                      # tile, chunk, jj, col, m, byte, half
            x = x.unflatten(-1, (-1, 4, 2))[..., _V4, :].transpose(-1, -2).flatten(-3, -2)
        else:
            x = x.unflatten(-1, (-1, 4))                           # tile, chunk, jj, col, n, r
        order = (n, n + 2, n + 5, n + 1, n + 4, n + 3)             # tile, jj, r, chunk, n, col
    else:
        x = x.unflatten(-1, (-1, 8))                               # tile, chunk, jj, t, kb, e
        if case["bits"] == 4:
            x = x[..., _K4]
        order = (n, n + 3, n + 1, n + 4, n + 2, n + 5)             # tile, t, chunk, kb, jj, e
    return x.permute(*range(n), *order).reshape(*lead, case["page"], -1)


def _cache_side(s, blocks, values):
    """K or V of head blocks [..., head bytes] in float32: [..., page, dim]."""
    _, groups, payload, meta = _geometry(s)
    x = _tokens(s, blocks[..., payload:2 * payload] if values else blocks[..., :payload], values)
    if not groups:
        return x.view(_DTYPES[s["dtype"]])[..., :s["dim"]].float()
    first = 2 * payload + (meta if values else 0)
    words = blocks[..., first:first + meta].contiguous().view(torch.float16).float()
    words = words.unflatten(-1, (s["page"], groups, 2))
    x = x.float().unflatten(-1, (-1, s["group"])) * words[..., :1] + words[..., 1:]
    return x.flatten(-2)[..., :s["dim"]]


def _plain_shared(s):
    b, hk, q = s["batch"], s["kv_heads"], s["queries"]
    blocks = s["pool"].unflatten(-1, (hk, -1))[s["table"].clamp_min(0).long()]       # [B, pages, HK, bytes]
    k, v = (_cache_side(s, blocks, side).transpose(1, 2).flatten(2, 3) for side in (False, True))
    rows = s["q"].float().reshape(b, hk, -1, s["dim"])
    scores = rows @ k.transpose(2, 3).contiguous() * s["dim"] ** -0.5
    last = s["lens"][:, None] - q + torch.arange(q, device="cuda")                   # each query's position
    last = last.repeat(1, s["heads"] // hk)[:, None, :, None]
    scores.masked_fill_(torch.arange(k.shape[2], device="cuda") > last, -math.inf)
    p = torch.exp(scores - scores.amax(-1, keepdim=True).clamp_min(-1e30))
    out = (p / p.sum(-1, keepdim=True).clamp_min(1e-30)) @ v.contiguous()
    return out.reshape(s["q"].shape).to(s["q"].dtype)


_PLAIN = {"rope": _plain_rope, "prompt": _plain_prompt, "shared": _plain_shared}


# ---- the same in 64 bits, from the definitions -----------------------------------------


def _exact_rope(s):
    h, hk, d, half = s["heads"], s["kv_heads"], s["dim"], _rotary(s) // 2
    x = s["qkv"].double().view(-1, h + 2 * hk, d).clone()
    starts, cached = s["starts"].tolist(), s["cached_lens"].tolist()
    for b, (lo, hi) in enumerate(zip(starts, starts[1:])):
        at = torch.arange(hi - lo, dtype=torch.float64, device="cuda") + cached[b]
        at = at[:, None].expand(-1, half)
        if "positions" in s:
            at = torch.stack([s["positions"][a, lo:hi].double() for a in s["axis"].tolist()], 1)
        # the pair as a complex number, turned by its angle
        z = torch.complex(x[lo:hi, :h + hk, :half], x[lo:hi, :h + hk, half:2 * half])
        z = z * torch.exp(1j * (at * s["inv_freq"].double()))[:, None]
        x[lo:hi, :h + hk, :half], x[lo:hi, :h + hk, half:2 * half] = z.real, z.imag
    out = {"q": x[:, :h], "pages": None}
    return dict(out, k=x[:, h:h + hk], v=x[:, h + hk:]) if s["with_kv"] else out


def _exact_prompt(s):
    h, hk = s["heads"], s["kv_heads"]
    out = torch.empty(s["q"].shape, dtype=torch.float64, device="cuda")
    starts = s["starts"].tolist()
    for lo, hi in zip(starts, starts[1:]):
        for first in range(lo, hi, 2048):
            last = min(hi, first + 2048)
            see = torch.arange(last - lo, device="cuda") <= torch.arange(first - lo, last - lo, device="cuda")[:, None]
            for i in range(h):
                k, v = (s[name][lo:last, i * hk // h].double() for name in "kv")
                x = s["q"][first:last, i].double() @ k.t().contiguous() / math.sqrt(s["dim"])
                out[first:last, i] = torch.softmax(x.masked_fill(~see, -math.inf), -1) @ v
    return out


def _exact_shared(s):
    gqa, page, hk, d = s["heads"] // s["kv_heads"], s["page"], s["kv_heads"], s["dim"]
    _, groups, payload, meta = _geometry(s)
    out = torch.empty(s["q"].shape, dtype=torch.float64, device="cuda")
    blocks = s["pool"].view(s["pool"].shape[0], hk, -1)
    for b, n in enumerate(s["lens"].tolist()):
        held = blocks[s["table"][b, :-(-n // page)].long()]
        sides = []
        for i in range(2):
            x = _tokens(s, held[..., i * payload:(i + 1) * payload], i == 1)
            if groups:
                words = held[..., 2 * payload + i * meta:2 * payload + (i + 1) * meta].contiguous()
                words = words.view(torch.float16).double().view(held.shape[0], hk, page, groups, 2)
                scale, bias = (words[..., j].repeat_interleave(s["group"], -1) for j in (0, 1))
                x = x.double() * scale + bias
            else:
                x = x.view(_DTYPES[s["dtype"]]).double()
            sides.append(x[..., :d].permute(1, 0, 2, 3).reshape(hk, -1, d)[:, :n].contiguous())
        k, v = sides
        for i in range(s["queries"]):
            see = n - s["queries"] + i + 1
            if see <= 0:
                out[b, :, i] = 0
                continue
            q = s["q"][b, :, i].double().view(hk, gqa, d)
            w = torch.softmax(torch.bmm(q, k[:, :see].transpose(1, 2).contiguous()) / math.sqrt(d), -1)
            out[b, :, i] = torch.bmm(w, v[:, :see].contiguous()).view(s["heads"], d)
    return out


def exact(case, seed):
    s = prepare(case, seed)
    return {"rope": _exact_rope, "prompt": _exact_prompt, "shared": _exact_shared}[case["kind"]](s)
