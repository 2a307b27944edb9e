"""What decides, on the device, which part of a paged cache lives on: the attention
weight that each cached token has drawn, eviction by it, and a beam step's selection
with the reordering of whatever the beams hold.

A case is a plain dict.  ``kind`` says which operator a pass runs:

* ``mass``    -- the attention weight that the queries of a step (or of the last
  stretch of a prompt) put on every cached token, summed over the query rows of each
  KV head and added to the sums so far.
* ``evict``   -- every (layer, sequence, KV head) keeps its first and last tokens and
  the heaviest of the others, up to a budget; the kept tokens' K and V move, in
  order, to pages of the sequence's own, their sums with them.
* ``beam``    -- log-softmax of the next token's logits, added to the beams' scores,
  and the best of all (beam, token) pairs of each group of beams.
* ``reorder`` -- each beam's rows of a state tensor become its parent's, all at once.

Where ``own`` is false a pass computes the operator in elementary torch operations
over the same tensors, the page layout's permutation among them; where it is true it
makes this package's calls.  Lengths are spread over ``lo..hi`` by a fixed rule, so a
case's sizes do not depend on the seed.
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

_DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32, "i32": torch.int32,
           "u8": torch.uint8}


def listed():
    return [
        # a small model on float pages: launches and host calls are all there is
        _mass("mass_bf16_small", batch=4, heads=8, kv_heads=2, dim=64, bits=16, lo=127, hi=511),
        # the serving step: 32 sequences of 1K..8K tokens on 8-bit pages, one query each
        _mass("mass_int8_b32", batch=32, lo=1024, hi=8191),
        # the last 32 queries of long prompts look back over 4-bit pages, eight heads per KV head
        _mass("mass_int4_window", batch=4, heads=32, kv_heads=4, page=32, bits=4, queries=32, lo=24000,
              hi=32767),
        # a few short chats on float pages halved
        _evict("evict_f16_small", batch=3, kv_heads=2, dim=64, bits=16, dtype="f16", lo=200, hi=500,
               keep=150),
        # a serving batch on 8-bit pages brought down to a budget of 1024 tokens
        _evict("evict_int8_b32", batch=32, lo=1024, hi=8191, keep=1024),
        # one long document, every layer of a small stack, a quarter kept
        _evict("evict_int4_long", layers=8, batch=1, kv_heads=4, page=32, bits=4, lo=32700, hi=32700,
               keep=8192),
        # one prompt, four beams, float logits
        _beam("beam_f32_small", batch=1, beams=4, vocab=32000, count=8, dtype="f32"),
        # a serving batch of beams over a large vocabulary
        _beam("beam_bf16_b32", batch=32, beams=4, vocab=128256, count=8),
        # many beams, rows of odd length, some hypotheses finished
        _beam("beam_f16_wide", batch=16, beams=16, vocab=49999, count=32, dtype="f16", finished=0.2),
        # the tokens of 32 hypotheses so far
        _reorder("reorder_tokens", dtype="i32", groups=8, beams=4, size=500),
        # the weight sums of 32 beams in 16 layers, into the other half of a double buffer
        _reorder("reorder_mass", dtype="f32", layers=16, groups=8, beams=4, size=8 * 2048, banks=2),
        # half-precision states of odd size, in place: a parent's first child stays where it is
        _reorder("reorder_states", dtype="bf16", layers=4, groups=16, beams=8, size=33333),
    ]


def _pages(kw):
    case = dict(batch=1, heads=32, kv_heads=8, dim=128, page=16, bits=8, group=64, dtype="bf16", lo=1024,
                hi=1024)
    case.update(kw)
    return case


def _mass(name, **kw):
    return dict(name=name, kind="mass", **_pages(dict(dict(queries=1), **kw)))


def _evict(name, **kw):
    kw = dict(dict(layers=1, sinks=4, recent=64), **kw)
    return dict(name=name, kind="evict", **_pages(kw))


def _beam(name, **kw):
    return dict(dict(name=name, kind="beam", dtype="bf16", finished=0.0), **kw)


def _reorder(name, **kw):
    return dict(dict(name=name, kind="reorder", layers=1, banks=1), **kw)


def _spread(rng, lo, hi):
    """A size of lo..hi, spread over its logarithm."""
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def _draw_pages(rng):
    dim = rng.choice([64, 128, 128, 128, 96, 80, 256])
    kv_heads = rng.choice([1, 2, 4, 8, 8])
    return dict(dim=dim, bits=rng.choice([8, 8, 4, 4, 16]), kv_heads=kv_heads,
                heads=kv_heads * rng.choice([1, 2, 4, 4, 7, 8]), page=rng.choice([16, 16, 32, 64, 128]),
                group=rng.choice([g for g in (32, 64, 128) if g <= max(64, dim // 2)]),
                dtype=rng.choice(["bf16", "bf16", "f16"]))


def draw(rng):
    most = max(_cost(c) for c in listed())
    while True:
        kind = rng.choice(["mass", "mass", "evict", "evict", "beam", "beam", "reorder"])
        if kind in ("mass", "evict"):
            lo = _spread(rng, 17, 24000)
            case = dict(kind=kind, batch=_spread(rng, 1, 48), lo=lo, hi=min(32767, lo + _spread(rng, 1, 2 * lo)),
                        **_draw_pages(rng))
            if kind == "mass":
                case["queries"] = rng.choice([1, 1, 1, rng.randint(2, 5), _spread(rng, 6, 64)])
            else:
                case.update(layers=rng.choice([1, 1, 2, 5]), keep=_spread(rng, 8, max(16, case["hi"])),
                            sinks=rng.randint(0, 8), recent=_spread(rng, 1, 200))
        elif kind == "beam":
            case = dict(kind=kind, batch=_spread(rng, 1, 64), beams=rng.randint(1, 16),
                        vocab=_spread(rng, 500, 200000), count=rng.randint(1, 40),
                        dtype=rng.choice(["bf16", "f16", "f32"]), finished=rng.choice([0.0, 0.0, 0.3]))
            case["count"] = min(case["count"], 2 * case["beams"])
        else:
            case = dict(kind=kind, dtype=rng.choice(["f32", "bf16", "i32", "u8"]), layers=rng.randint(1, 16),
                        groups=_spread(rng, 1, 32), beams=rng.randint(2, 16), size=_spread(rng, 16, 100000),
                        banks=rng.choice([1, 2]))
        if _cost(case) <= 0.8 * most and _held(case) <= 1.2e9:
            return case


# ---- sizes -------------------------------------------------------------------------


def _lengths(case):
    """Tokens per sequence."""
    n, lo, hi = case["batch"], case["lo"], case["hi"]
    return [lo + int((hi - lo) * ((i + 1) * 0.6180339887498949 % 1.0)) if n > 1 else hi for i in range(n)]


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


def _parents(beams):
    return (beams + 1) // 2


def _element(case):
    return torch.empty(0, dtype=_DTYPES[case["dtype"]]).element_size()


def work(case):
    if case["kind"] == "reorder":
        moved = case["beams"] if case["banks"] == 2 else case["beams"] - _parents(case["beams"])
        rows = case["layers"] * case["groups"] * moved
        return {"bytes": 2 * rows * case["size"] * _element(case), "flops": 0}
    if case["kind"] == "beam":
        rows = case["batch"] * case["beams"]
        live = rows - rows * case["finished"]
        return {"bytes": live * case["vocab"] * _element(case) + 12 * case["batch"] * case["count"],
                "flops": 3 * live * case["vocab"]}
    lengths, hk = _lengths(case), case["kv_heads"]
    if case["kind"] == "evict":
        kept = sum(min(n, case["keep"]) for n in lengths)
        # the sums read; the kept tokens' sums, indices, K and V written, K and V read
        return {"bytes": case["layers"] * hk * (4 * sum(lengths) + kept * (8 + 4 * _side_bytes(case))), "flops": 0}
    rows = case["batch"] * case["heads"] * case["queries"]
    # K and the sums read, the sums written, the queries read
    nbytes = sum(lengths) * hk * (_side_bytes(case) + 8) + 2 * rows * case["dim"]
    q = case["queries"]
    pairs = case["heads"] * sum(q * n - q * (q - 1) // 2 if n >= q else n * (n + 1) // 2 for n in lengths)
    return {"bytes": nbytes, "flops": 2 * case["dim"] * pairs}


def _cost(case):
    w = work(case)
    return max(w["bytes"], w["flops"] / 50)


def _held(case):
    """Bytes that a state holds, roughly."""
    if case["kind"] in ("mass", "evict"):
        dp, _, payload, meta = _geometry(case)
        tokens = case["batch"] * (case["hi"] + case.get("keep", 0))
        return case.get("layers", 1) * tokens * case["kv_heads"] * 2 * (payload + meta) / case["page"]
    return (8 if case["kind"] == "beam" else 2) * work(case)["bytes"]


# ---- inputs ------------------------------------------------------------------------


def _generator(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(int(seed) * 7919 + 29)
    return g


def _ints(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def _tables(case, counts, seed):
    """Block tables (one per list of pages per sequence) over one set of shuffled page ids."""
    total = sum(sum(c) for c in counts)
    ids = np.random.default_rng(seed).permutation(total).astype(np.int32)
    at, tables = 0, []
    for c in counts:
        c = np.asarray(c)
        table = np.full((len(c), max(int(c.max()), 1)), -1, np.int32)
        place = np.arange(table.shape[1])[None, :] < c[:, None]
        table[place] = ids[at:at + int(c.sum())]
        at += int(c.sum())
        tables.append(torch.from_numpy(table).cuda())
    return tables, max(total, 1)


def _quantized(case, x):
    """Codes [..., dp] u8 and (scale, bias) words [..., groups] of rows x [..., dp]."""
    levels = float(2 ** case["bits"] - 1)
    x = x.float().unflatten(-1, (-1, case["group"]))
    low = x.amin(-1, keepdim=True).half()
    step = ((x.amax(-1, keepdim=True) - low.float()) / levels).clamp_min(1e-6).half()
    codes = ((x - low.float()) / step.float()).round().clamp(0, levels).to(torch.uint8).flatten(-2)
    words = torch.stack((step, low), -1).squeeze(-2).contiguous().view(torch.int32).squeeze(-1)
    return codes, words


def _rows(case, gen, shape):
    """K or V rows N(0, 1), padded with zeros to the stored dim, a few head-dim channels larger, as
    a page side holds them: (elements, metadata words or None)."""
    dp = _geometry(case)[0]
    x = torch.randn(shape + (case["dim"],), generator=gen, device="cuda")
    gain = torch.ones(case["dim"], device="cuda")
    gain[torch.randperm(case["dim"], generator=gen, device="cuda")[:2]] = 3.0
    x = torch.nn.functional.pad((x * gain).to(_DTYPES[case["dtype"]]), (0, dp - case["dim"]))
    return (x.view(torch.int16), None) if case["bits"] == 16 else _quantized(case, x)


def _pool(case, gen, pages):
    """A layer's pool of `pages` filled pages, [pages, page bytes] u8."""
    shape = (pages, case["kv_heads"], case["page"])
    return _join(case, _rows(case, gen, shape), _rows(case, gen, shape)).flatten(1)


# The page layout: a head block is the K tiles, the V tiles (16 tokens each), then for quantized pages the
# K and V metadata words.  A tile is `chunks` chunks of 64 lanes of `cs` bytes; K's lane 16*jj + t holds
# dims 32*kb + 8*jj + e of token t, V's lane 16*jj + c holds tokens 4*jj + r of dims 16*n + c.


def _chunks(case):
    lane = _geometry(case)[0] * case["bits"] // 32
    cs = min(16, lane)
    return lane // cs, cs


def _elements(case, payload):
    """Lane bytes [..., cs] as elements in the lane's order: int16, u8, or a nibble per u8."""
    if case["bits"] == 16:
        return payload.view(torch.int16)
    return payload if case["bits"] == 8 else torch.stack((payload & 15, payload >> 4), -1).flatten(-2)


def _lane_bytes(case, x):
    if case["bits"] == 16:
        return x.contiguous().view(torch.uint8)
    x = x.contiguous()
    return x if case["bits"] == 8 else x[..., 0::2] | (x[..., 1::2] << 4)


_K4 = [0, 4, 1, 5, 2, 6, 3, 7]  # the nibble of a K word's element e
_V4 = [0, 2, 1, 3]              # the byte of a V word's token r


def _k_side(case, payload):
    """K payload bytes [..., payload] -> elements [..., page, dp]."""
    nch, cs = _chunks(case)
    lead = payload.shape[:-1]
    x = _elements(case, payload.reshape(*lead, -1, nch, 4, 16, cs))
    x = x.unflatten(-1, (-1, 8))                                   # tile, chunk, jj, t, kb, e
    if case["bits"] == 4:
        x = x[..., _K4]
    n = len(lead)
    x = x.permute(*range(n), n, n + 3, n + 1, n + 4, n + 2, n + 5)  # tile, t, chunk, kb, jj, e
    return x.reshape(*lead, case["page"], -1)


def _k_payload(case, x):
    nch, cs = _chunks(case)
    lead, n = x.shape[:-2], x.dim() - 2
    x = x.reshape(*lead, case["page"] // 16, 16, nch, cs // case["bits"], 4, 8)
    x = x.permute(*range(n), n, n + 2, n + 4, n + 1, n + 3, n + 5)
    if case["bits"] == 4:
        x = x[..., torch.argsort(torch.tensor(_K4)).tolist()]
    return _lane_bytes(case, x.flatten(-2)).reshape(*lead, -1)


def _v_side(case, payload):
    """V payload bytes [..., payload] -> elements [..., page, dp]."""
    nch, cs = _chunks(case)
    lead = payload.shape[:-1]
    n = len(lead)
    x = _elements(case, payload.reshape(*lead, -1, nch, 4, 16, cs))
    if case["bits"] == 4:                                          # tile, chunk, jj, col, m, byte, half
        x = x.unflatten(-1, (-1, 4, 2))[..., _V4, :].transpose(-1, -2).flatten(-3, -2)
    else:
        x = x.unflatten(-1, (-1, 4))                               # tile, chunk, jj, col, n, r
    x = x.permute(*range(n), n, n + 2, n + 5, n + 1, n + 4, n + 3)  # tile, jj, r, chunk, n, col
    return x.reshape(*lead, case["page"], -1)


def _v_payload(case, x):
    nch, cs = _chunks(case)
    lead, n = x.shape[:-2], x.dim() - 2
    per = cs * 8 // case["bits"] // 4                              # blocks of 16 dims per chunk
    x = x.reshape(*lead, case["page"] // 16, 4, 4, nch, per, 16)
    x = x.permute(*range(n), n, n + 3, n + 1, n + 5, n + 4, n + 2)
    if case["bits"] == 4:
        x = x.unflatten(-2, (-1, 2)).transpose(-1, -2)[..., _V4, :].flatten(-3)
    else:
        x = x.flatten(-2)
    return _lane_bytes(case, x).reshape(*lead, -1)


def _split(case, heads, values=True):
    """Head blocks [..., head bytes] -> ((K elements, K words), (V elements, V words))."""
    _, groups, payload, meta = _geometry(case)
    sides = []
    for at, form in ((0, _k_side), (1, _v_side))[:2 if values else 1]:
        words = None
        if groups:
            words = heads[..., 2 * payload + at * meta:2 * payload + (at + 1) * meta].contiguous()
            words = words.view(torch.int32).unflatten(-1, (case["page"], groups))
        sides.append((form(case, heads[..., at * payload:(at + 1) * payload]), words))
    return sides


def _join(case, k, v):
    """The inverse: head blocks [..., head bytes] u8."""
    parts = [_k_payload(case, k[0]), _v_payload(case, v[0])]
    if k[1] is not None:
        parts += [w.contiguous().view(torch.uint8).flatten(-2) for w in (k[1], v[1])]
    return torch.cat(parts, -1)


def _weights_so_far(gen, shape):
    """Accumulated attention weight of a few steps: most tokens hardly any, a few a great deal."""
    return torch.empty(shape, device="cuda").exponential_(generator=gen).pow_(3) * 1e-3


def prepare(case, seed):
    gen = _generator(seed)
    s = dict(case)
    if case["kind"] == "mass":
        lengths = _lengths(case)
        (s["table"],), pages = _tables(case, [[-(-n // case["page"]) for n in lengths]], seed)
        s["pool"] = _pool(case, gen, pages)
        s["lens"] = _ints(lengths)
        s["counted"] = s["lens"] - case["queries"]  # the step's own tokens have no sum yet
        s["q"] = torch.randn((case["batch"], case["heads"], case["queries"], case["dim"]), generator=gen,
                             device="cuda").to(_DTYPES[case["dtype"]])
        shape = (case["batch"] + 2, case["kv_heads"], s["table"].shape[1] * case["page"])
        s["mass"] = _weights_so_far(gen, shape)
        s["rows"] = torch.randperm(shape[0], generator=gen, device="cuda")[:case["batch"]].to(torch.int32)
        s["out"] = torch.zeros(shape, device="cuda")
    elif case["kind"] == "evict":
        lengths = _lengths(case)
        page = case["page"]
        tables, pages = _tables(case, [[-(-n // page) for n in lengths],
                                       [-(-min(n, case["keep"]) // page) for n in lengths]], seed)
        s["src"], s["dst"] = tables
        s["pools"] = torch.stack([_pool(case, gen, pages) for _ in range(case["layers"])])
        s["lens"] = _ints(lengths)
        s["mass"] = _weights_so_far(gen, (case["layers"], case["batch"], case["kv_heads"],
                                          s["src"].shape[1] * page))
    elif case["kind"] == "beam":
        # as a language model's: a few tokens far above a broad floor
        shape = (case["batch"], case["beams"], case["vocab"])
        x = torch.randn(shape, generator=gen, device="cuda")
        s["logits"] = (2.5 * x + 0.25 * x.pow(3)).to(_DTYPES[case["dtype"]])
        s["scores"] = -torch.rand(shape[:2], generator=gen, device="cuda") * 20
        s["done"] = torch.rand(shape[:2], generator=gen, device="cuda") < case["finished"]
        s["done"][:, 0] = False
    else:
        beams, groups = case["beams"], case["groups"]
        shape = (case["layers"], case["banks"] * groups * beams, case["size"])
        dtype = _DTYPES[case["dtype"]]
        s["state"] = (torch.randn(shape, generator=gen, device="cuda").to(dtype) if dtype.is_floating_point
                      else torch.randint(0, 250, shape, generator=gen, device="cuda", dtype=dtype))
        parents = torch.randint(0, beams, (groups, beams), generator=gen, device="cuda")
        if case["banks"] == 1:  # in place: the parents keep their places, their other children take the rest
            order = torch.rand((groups, beams), generator=gen, device="cuda").argsort(1)
            parents.scatter_(1, order, order[:, torch.arange(beams, device="cuda") % _parents(beams)])
        first = torch.arange(groups, device="cuda")[:, None] * beams
        s["sources"] = (first + parents).flatten().to(torch.int32)
        s["targets"] = torch.arange(groups * beams, dtype=torch.int32, device="cuda")
        s["targets"] += (case["banks"] - 1) * groups * beams
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


def _own_mass(s):
    from pkv import ops

    return ops.attention_mass(_format(s), s["pool"], s["q"], s["table"], s["lens"], scale=s["dim"] ** -0.5,
                              mass=s["mass"], counted=s["counted"], rows=s["rows"], out=s["out"])


def _own_evict(s):
    from pkv import ops

    kept, lens, mass = ops.evict_select(s["mass"], s["lens"], s["keep"], sinks=s["sinks"], recent=s["recent"],
                                        with_mass=True)
    ops.evict_pages(_format(s), s["pools"], kept, lens, s["src"], s["dst"])
    return {"kept": kept, "lens": lens, "mass": mass, "pages": s["pools"]}


def _own_beam(s):
    from pkv import ops

    scores, parents, tokens = ops.beam_select(s["logits"], s["scores"], s["count"], done=s["done"], pad_token=0)
    return {"scores": scores, "parents": parents, "tokens": tokens}


def _own_reorder(s):
    from pkv import ops

    ops.reorder_rows(s["state"], s["targets"], s["sources"], dim=1)
    return s["state"]


_OWN = {"mass": _own_mass, "evict": _own_evict, "beam": _own_beam, "reorder": _own_reorder}


def _plain_mass(s):
    b, hk, q = s["batch"], s["kv_heads"], s["queries"]
    heads = s["pool"].unflatten(-1, (hk, -1))[s["table"].clamp_min(0).long()]        # [B, pages, HK, bytes]
    ((k, words),) = _split(s, heads, values=False)
    if words is not None:
        words = words.view(torch.float16).float().unflatten(-1, (-1, 2))
        k = (k.float().unflatten(-1, (-1, s["group"])) * words[..., :1] + words[..., 1:]).flatten(-2)
    else:
        k = k.view(_DTYPES[s["dtype"]]).float()
    k = k[..., :s["dim"]].transpose(1, 2).flatten(2, 3)                              # [B, HK, T, D]
    rows = s["q"].float().reshape(b, hk, -1, s["dim"])
    scores = rows @ k.transpose(2, 3).contiguous() * s["dim"] ** -0.5
    last = s["lens"][:, None] - q + torch.arange(q, device="cuda")                   # each query's position
    last = last.repeat(1, s["heads"] // hk)[:, None, :, None]
    t = torch.arange(k.shape[2], device="cuda")
    scores.masked_fill_(t > last, -math.inf)
    p = torch.exp(scores - scores.amax(-1, keepdim=True).clamp_min(-1e30))
    new = (p / p.sum(-1, keepdim=True).clamp_min(1e-30)).sum(2)                      # 0 where a query sees nothing
    at = s["rows"].long()
    old = torch.where(t < s["counted"][:, None, None], s["mass"][at], torch.zeros_like(new))
    s["out"][at] = torch.where(t < s["lens"][:, None, None], old + new, s["out"][at])
    return s["out"]


def _plain_evict(s):
    mass, lens, top = s["mass"], s["lens"].long(), s["keep"]
    t = torch.arange(mass.shape[-1], device="cuda")
    n = lens.clamp_max(top)
    recent = n.clamp_max(s["recent"])
    sinks = torch.minimum(n - recent, torch.full_like(n, s["sinks"]))
    lens_, n_, recent_, sinks_ = (x[:, None, None] for x in (lens, n, recent, sinks))
    key = mass.masked_fill((t < sinks_) | (t >= lens_ - recent_), math.inf).masked_fill(t >= lens_, -math.inf)
    order = torch.sort(key, dim=-1, descending=True, stable=True).indices            # ties: the lowest index first
    taken = order.masked_fill(t >= n_, mass.shape[-1])                               # the heaviest n
    kept = torch.sort(taken, dim=-1).values[..., :top]
    kept = torch.nn.functional.pad(kept, (0, top - kept.shape[-1]), value=mass.shape[-1])
    place = torch.arange(top, device="cuda")
    live = place < n_
    index = kept.clamp_max(mass.shape[-1] - 1)
    new_mass = mass.gather(-1, index) * live
    src, dst = s["src"].clamp_min(0).long(), s["dst"].clamp_min(0).long()
    heads = s["pools"].unflatten(-1, (s["kv_heads"], -1))
    stay = _split(s, heads[:, dst])
    sides = []
    width = s["dst"].shape[1] * s["page"]
    index, live = (torch.nn.functional.pad(x, (0, max(0, width - top)))[..., :width] for x in (index, live))
    for (old, old_words), (here, here_words) in zip(_split(s, heads[:, src]), stay):
        new = []
        for x, y in ((old, here), (old_words, here_words)):
            if x is None:
                new.append(None)
                continue
            tokens, held = (z.transpose(2, 3).flatten(3, 4) for z in (x, y))         # [L, B, HK, T, values]
            tokens = tokens.gather(3, index[..., None].expand(*index.shape, tokens.shape[-1]))
            tokens = torch.where(live[..., None], tokens, held)
            new.append(tokens.unflatten(3, (-1, s["page"])).transpose(2, 3))
        sides.append(new)
    mapped = (s["dst"] >= 0)
    heads[:, dst[mapped]] = _join(s, *sides)[:, mapped]
    kept = kept.masked_fill(~(place < n_), -1).to(torch.int32)
    return {"kept": kept, "lens": n.to(torch.int32), "mass": new_mass, "pages": s["pools"]}


def _plain_beam(s):
    # in 64 bits: which of two beams' tokens comes first hangs on their last digits
    x = s["logits"].double()
    x = x - x.amax(-1, keepdim=True)
    x = x - torch.log(torch.exp(x).sum(-1, keepdim=True)) + s["scores"].double()[..., None]
    finished = torch.full_like(x, -math.inf)
    finished[..., 0] = s["scores"].double()
    x = torch.where(s["done"][..., None], finished, x).flatten(1)
    best = torch.sort(x, dim=-1, descending=True, stable=True)
    scores, flat = best.values[:, :s["count"]], best.indices[:, :s["count"]]
    return {"scores": scores.float(), "parents": (flat // s["vocab"]).to(torch.int32),
            "tokens": (flat % s["vocab"]).to(torch.int32)}


def _plain_reorder(s):
    s["state"][:, s["targets"].long()] = s["state"][:, s["sources"].long()]
    return s["state"]


_PLAIN = {"mass": _plain_mass, "evict": _plain_evict, "beam": _plain_beam, "reorder": _plain_reorder}


# ---- the same in 64 bits, from the definitions -----------------------------------------


def _exact_mass(s):
    out = torch.zeros(s["mass"].shape, dtype=torch.float64, device="cuda")
    gqa, page = s["heads"] // s["kv_heads"], s["page"]
    _, groups, payload, meta = _geometry(s)
    blocks = s["pool"].view(s["pool"].shape[0], s["kv_heads"], -1)
    for b, n in enumerate(s["lens"].tolist()):
        pages = s["table"][b, :-(-n // page)].long()
        k = _k_side(s, blocks[pages][..., :payload])
        if groups:
            meta_b = blocks[pages][..., 2 * payload:2 * payload + meta].contiguous().view(torch.float16).double()
            meta_b = meta_b.view(len(pages), s["kv_heads"], page, groups, 2)
            scale, bias = (meta_b[..., i].repeat_interleave(s["group"], -1) for i in (0, 1))
            k = k.double() * scale + bias
        else:
            k = k.view(_DTYPES[s["dtype"]]).double()
        k = k[..., :s["dim"]].permute(1, 0, 2, 3).reshape(s["kv_heads"], -1, s["dim"])[:, :n].contiguous()
        total = torch.zeros((s["kv_heads"], n), dtype=torch.float64, device="cuda")
        for i in range(s["queries"]):
            see = n - s["queries"] + i + 1
            if see > 0:
                q = s["q"][b, :, i].double().view(s["kv_heads"], gqa, s["dim"])
                w = torch.softmax(torch.bmm(q, k[:, :see].transpose(1, 2).contiguous()) / math.sqrt(s["dim"]), -1)
                total[:, :see] += w.sum(1)
        row, old = int(s["rows"][b]), max(0, n - s["queries"])
        total[:, :old] += s["mass"][row, :, :old].double()
        out[row, :, :n] = total
    return out


def exact(case, seed):
    s = prepare(case, seed)
    if case["kind"] == "mass":
        return _exact_mass(s)
    if case["kind"] == "beam":
        rows = torch.log_softmax(s["logits"].double(), -1) + s["scores"].double()[..., None]
        rows[s["done"]] = -math.inf
        rows[..., 0] = torch.where(s["done"], s["scores"].double(), rows[..., 0])
        best = torch.topk(rows.flatten(1), case["count"], dim=-1).values
        return {"scores": best, "parents": None, "tokens": None}
    if case["kind"] == "evict":
        # the sums of the kept tokens, by threshold instead of by order
        n = s["lens"].long().clamp_max(case["keep"])
        out = torch.zeros((case["layers"], case["batch"], case["kv_heads"], case["keep"]), dtype=torch.float64,
                          device="cuda")
        for b, (length, most) in enumerate(zip(s["lens"].tolist(), n.tolist())):
            last = min(case["recent"], most)
            first = min(case["sinks"], most - last)
            m = s["mass"][:, b, :, :length].double()
            middle = m[..., first:length - last]
            need = most - first - last
            stays = torch.ones_like(m, dtype=torch.bool)
            stays[..., first:length - last] = False
            if need:
                least = torch.kthvalue(middle, middle.shape[-1] - need + 1, dim=-1, keepdim=True).values
                above = middle > least
                level = middle == least
                room = need - above.sum(-1, keepdim=True)
                stays[..., first:length - last] = above | (level & (level.cumsum(-1) <= room))
            out[:, b, :, :most] = m[stays].view(case["layers"], case["kv_heads"], most)
        return {"kept": None, "lens": None, "mass": out, "pages": None}
    if _DTYPES[case["dtype"]].is_floating_point:
        out = s["state"].double().clone()
        for target, source in zip(s["targets"].tolist(), s["sources"].tolist()):
            out[:, target] = s["state"][:, source].double()
        return out
    return None
