"""Cases of the paged-cache operators: appending rotated keys and values to a
paged cache (bf16, or E4M3 with one power-of-two scale per page and head) and
attention over that cache, for one token per sequence up to whole prompts.

``run`` computes an operator in plain torch (32-bit arithmetic, one rounding at
the end) or, with ``own`` set, through ``thor_megakernels_b200.paged``.
"""
import math
import random

import torch

own = False

E4M3_MAX = 448.0
SCALE_EXPONENTS = (-64, 120)   # range of the exponent of a page's scale
BF16, E4M3 = "bf16", "e4m3"
CACHE_TYPES = {BF16: torch.bfloat16, E4M3: torch.float8_e4m3fn}


def _append(name, cache, heads, kv_heads, dim, page, seqs, new, start, rot=None, layout="interleaved"):
    """``new``: tokens a sequence gets, or "a-b" for ragged counts in that range; ``start``: cached positions before, likewise."""
    return dict(name=name, op="append", cache=cache, heads=heads, kv_heads=kv_heads, dim=dim, page=page, seqs=seqs, new=str(new),
                start=str(start), rot=rot or dim, layout=layout)


def _attention(name, cache, heads, kv_heads, dim, page, seqs, new, start, empty=0):
    """``empty``: the first so many sequences hold nothing (padding slots of a captured batch)."""
    return dict(name=name, op="attention", cache=cache, heads=heads, kv_heads=kv_heads, dim=dim, page=page, seqs=seqs, new=str(new),
                start=str(start), empty=empty)


def listed():
    return [
        # one sequence decoding by itself: a single row to rotate and store, nothing but latency
        _append("append 1 row bf16", BF16, 32, 8, 128, 16, 1, 1, 115),
        # a full decode batch over an 8-bit cache: every page's scale may have to grow
        _append("append 128 rows e4m3", E4M3, 32, 8, 128, 64, 128, 1, "64-1023", layout="half"),
        # verification of drafted tokens on one shard of a split model, rotary part of the head only
        _append("append 33x5 rows e4m3", E4M3, 16, 4, 64, 32, 33, 5, "0-2000", rot=32),
        # a prompt chunk on the same shard, bf16 cache
        _append("append 2 prompts bf16", BF16, 16, 4, 64, 64, 2, "900-1100", 0),
        # ragged prompts admitted together, 8-bit cache: bandwidth
        _append("append 7 prompts e4m3", E4M3, 32, 8, 128, 64, 7, "601-2100", "0-300", layout="half"),
        # the headline request: one sequence, about a hundred cached positions
        _attention("decode 1x116 bf16", BF16, 32, 8, 64, 16, 1, 1, 115),
        # one long conversation decoded alone: the long axis has to be split
        _attention("decode 1x65521 e4m3", E4M3, 32, 8, 128, 64, 1, 1, 65520),
        # a moderate batch with an idle slot, bf16 cache
        _attention("decode 17x4096 bf16", BF16, 32, 8, 128, 32, 17, 1, "511-4095", empty=1),
        # a full batch over the 8-bit cache
        _attention("decode 128x4096 e4m3", E4M3, 32, 8, 128, 64, 128, 1, "511-4095"),
        # drafted tokens verified five at a time, small pages
        _attention("verify 32x5 e4m3", E4M3, 16, 4, 64, 16, 32, 5, "0-2000"),
        # a chunk of a long prompt behind what is cached already
        _attention("chunk 512 at 8192 e4m3", E4M3, 32, 8, 128, 64, 1, 512, 8192),
        # whole prompts of different lengths
        _attention("4 prompts bf16", BF16, 32, 8, 128, 64, 4, "333-3001", 0),
    ]


def _log_int(rng, low, high):
    return min(high, int(low * math.exp(rng.random() * math.log((high + 1) / low))))


def draw(rng):
    cache, dim, page = rng.choice((BF16, E4M3)), rng.choice((64, 128)), rng.choice((16, 32, 64, 128))
    kv_heads = rng.choice((1, 2, 4, 8))
    heads = kv_heads * rng.choice((1, 2, 4, 4, 7, 8))
    kind = rng.choice(("append rows", "append prompts", "decode", "decode", "verify", "prompts"))
    if kind == "append rows":
        c = _append("", cache, heads, kv_heads, dim, page, _log_int(rng, 1, 256), rng.randint(1, 8), "0-%d" % _log_int(rng, 16, 4000),
                    rot=rng.choice((dim, dim, dim // 2, dim // 4)), layout=rng.choice(("interleaved", "half")))
    elif kind == "append prompts":
        n = _log_int(rng, 30, 2000)
        c = _append("", cache, heads, kv_heads, dim, page, rng.randint(1, 5), "%d-%d" % (n // 2 + 1, n), "0-%d" % rng.choice((0, 300)),
                    rot=rng.choice((dim, dim, dim // 2)), layout=rng.choice(("interleaved", "half")))
    elif kind in ("decode", "verify"):
        seqs = _log_int(rng, 1, 96)
        c = _attention("", cache, heads, kv_heads, dim, page, seqs, 1 if kind == "decode" else rng.randint(2, 9),
                       "0-%d" % _log_int(rng, 20, min(60000, 240000 // seqs)), empty=rng.choice((0, 0, 1)) if seqs > 1 else 0)
    else:
        n = _log_int(rng, 20, 1500)
        c = _attention("", cache, heads, kv_heads, dim, page, rng.randint(1, 4), "%d-%d" % (n // 2 + 1, n), "0-%d" % rng.choice((0, 700, 4000)))
    del c["name"]
    while True:   # never more than the largest listed cases
        w = work(c)
        if w["bytes"] <= 6e8 and w["flops"] <= 1.2e11:
            return c
        c["seqs"], c["start"] = max(1, c["seqs"] * 3 // 4), "0-%d" % (int(c["start"].partition("-")[2]) * 3 // 4)


def _between(text, rng):
    low, _, high = text.partition("-")
    return rng.randint(int(low), int(high or low))


def _lengths(case):
    """(new tokens, cached positions before them) of every sequence, from the case alone."""
    rng = random.Random(17)
    new = [_between(case["new"], rng) for _ in range(case["seqs"])]
    start = [_between(case["start"], rng) for _ in range(case["seqs"])]
    for text, values in ((case["new"], new), (case["start"], start)):   # the upper end is always met
        if values:
            values[-1] = int(text.partition("-")[2] or text)
    if case["op"] == "attention":
        start[:case["empty"]] = [0] * case["empty"]
    return new, start


def _scale_for(amax):
    """The smallest power-of-two scale that brings ``amax`` into E4M3's range."""
    mantissa, exponent = torch.frexp(amax)
    e = torch.where(mantissa <= E4M3_MAX / 512, exponent - 9, exponent - 8)
    e = torch.where(amax > 0, e, SCALE_EXPONENTS[0]).clamp(*SCALE_EXPONENTS)
    return torch.exp2(e.double()).float()


def _take(pages, at):
    """Chosen pages as 32-bit values (8-bit types are indexed as bytes)."""
    return pages[at].float() if pages.dtype == torch.bfloat16 else pages.view(torch.uint8)[at].view(pages.dtype).float()


def _pages(case, count, gen):
    """Page pools as earlier steps left them: keys, values and (8-bit) their scales; every page has its own magnitude."""
    shape = (count, case["kv_heads"], case["page"], case["dim"])
    out = []
    for _ in range(2):
        x = torch.randn(shape, generator=gen, device="cuda")
        x *= torch.exp2(torch.randn((count, case["kv_heads"], 1, 1), generator=gen, device="cuda"))
        if case["cache"] == BF16:
            out.append((x.bfloat16(), None))
        else:
            scale = _scale_for(x.abs().amax(dim=(2, 3)))
            out.append(((x / scale[:, :, None, None]).to(torch.float8_e4m3fn), scale))
    return out


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    new, start = _lengths(case)
    page, dim, heads, kv_heads = case["page"], case["dim"], case["heads"], case["kv_heads"]
    need = [-(-(n + s) // page) for n, s in zip(new, start)]
    columns, total = max(need), sum(need)
    order = torch.randperm(total + 3, generator=gen, device="cuda").int()
    table = torch.full((case["seqs"], columns), -1, dtype=torch.int32)
    at = torch.arange(total, dtype=torch.int32).split(need)
    for b, pages in enumerate(at):
        table[b, :len(pages)] = pages
    table = torch.where(table.cuda() >= 0, order[table.cuda().clamp(min=0).long()], -1).int().contiguous()
    (k, k_scales), (v, v_scales) = _pages(case, total + 3, gen)
    tokens = sum(new)
    cu = torch.tensor([0] + new, dtype=torch.int32).cumsum(0).int().cuda()
    ragged = len(set(new)) > 1
    s = dict(op=case["op"], k_pages=k, v_pages=v, k_scales=k_scales, v_scales=v_scales, page_table=table, cu_tokens=cu if ragged else None,
             page=page, most_new=max(new))
    if case["op"] == "append":
        # what a fused projection leaves: q, k and v side by side in one panel
        panel = torch.randn((tokens, (heads + 2 * kv_heads) * dim), generator=gen, device="cuda") * 1.5
        panel = panel.bfloat16()
        s["q"], s["k"], s["v"] = (x.unflatten(1, (-1, dim)) for x in panel.split((heads * dim, kv_heads * dim, kv_heads * dim), dim=1))
        s["start"] = torch.tensor(start, dtype=torch.int32).cuda()
        s["rope_cos"], s["rope_sin"] = _tables(case["rot"], max(n + p for n, p in zip(new, start)), case["layout"])
        s["layout"] = case["layout"]
    else:
        s["q"] = (torch.randn((tokens, heads, dim), generator=gen, device="cuda") * 2).bfloat16()
        lengths = [n + p for n, p in zip(new, start)]
        lengths[:case["empty"]] = [0] * case["empty"]
        s["lengths"] = torch.tensor(lengths, dtype=torch.int32).cuda()
        s["scale"] = 1 / math.sqrt(dim)
    return s


def _tables(rot, positions, layout):
    """Rotary tables as a model keeps them: fp32 [positions, rot], one column per element."""
    inv = 500000.0 ** (-torch.arange(0, rot, 2, dtype=torch.float64, device="cuda") / rot)
    angle = torch.arange(positions, dtype=torch.float64, device="cuda")[:, None] * inv
    angle = torch.cat((angle, angle), dim=1) if layout == "half" else angle.repeat_interleave(2, dim=1)
    return angle.cos().float(), angle.sin().float()


def run(s):
    if own:
        from thor_megakernels_b200 import paged

        cache = (s["k_pages"], s["v_pages"])
        scales = dict(k_scales=s["k_scales"], v_scales=s["v_scales"])
        if s["op"] == "append":
            q = paged.append(s["k"], s["v"], *cache, s["page_table"], s["start"], q=s["q"], rope_cos=s["rope_cos"], rope_sin=s["rope_sin"],
                             layout=s["layout"], cu_tokens=s["cu_tokens"], **scales)
            return dict(q=q, k_pages=s["k_pages"], v_pages=s["v_pages"], **scales)
        return paged.attention(s["q"], *cache, s["page_table"], s["lengths"], scale=s["scale"], cu_tokens=s["cu_tokens"], **scales)
    return _plain_append(s) if s["op"] == "append" else _plain_attention(s)


def _rotate(x, cos, sin, layout):
    """x [tokens, heads, dim] in 32 bits; the first ``cos.shape[1]`` elements of a head are rotated."""
    rot = cos.shape[1]
    head, rest = x[..., :rot], x[..., rot:]
    if layout == "half":
        other = torch.cat((-head[..., rot // 2:], head[..., :rot // 2]), dim=-1)
    else:
        other = torch.stack((-head[..., 1::2], head[..., 0::2]), dim=-1).flatten(-2)
    return torch.cat((head * cos[:, None] + other * sin[:, None], rest), dim=-1)


def _sequence_of(s, tokens, seqs):
    """(sequence, index within its new tokens) of every row."""
    row = torch.arange(tokens, device=s["q"].device)
    if s["cu_tokens"] is None:
        return row // (tokens // seqs), row % (tokens // seqs)
    b = torch.searchsorted(s["cu_tokens"], row.int(), right=True) - 1
    return b, row - s["cu_tokens"][b]


def _plain_append(s):
    tokens, page = s["q"].shape[0], s["page"]
    b, i = _sequence_of(s, tokens, s["start"].shape[0])
    pos = s["start"][b] + i
    cos, sin = s["rope_cos"][pos], s["rope_sin"][pos]
    q = _rotate(s["q"].float(), cos, sin, s["layout"]).bfloat16()
    at, slot = s["page_table"][b, pos // page].long(), (pos % page).long()
    for x, pages, scales in ((_rotate(s["k"].float(), cos, sin, s["layout"]), s["k_pages"], s["k_scales"]),
                             (s["v"].float(), s["v_pages"], s["v_scales"])):
        if scales is None:
            pages[at, :, slot] = x.to(pages.dtype)
        else:
            _plain_store(x, pages, scales, at, slot, s)
    return dict(q=q, k_pages=s["k_pages"], v_pages=s["v_pages"], k_scales=s["k_scales"], v_scales=s["v_scales"])


def _plain_store(x, pages, scales, at, slot, s):
    """The 8-bit cache: a page's scale grows to fit the new rows, and rows that the page held already are coded anew."""
    start, page = s["start"], s["page"]
    held = (start % page).long()                                                 # rows that a sequence's first page holds
    first = s["page_table"].gather(1, (start // page).clamp(max=s["page_table"].shape[1] - 1)[:, None].long())[:, 0]
    held = torch.where(first >= 0, held, 0)
    first = first.clamp(min=0).long()
    amax = torch.zeros_like(scales).index_reduce_(0, at, x.abs().amax(dim=-1), "amax")
    fit = _scale_for(amax)
    old = scales[first]
    grown = torch.where(held[:, None] > 0, torch.maximum(old, fit[first]), fit[first])
    fit = fit.index_copy(0, first, grown)
    codes = _take(pages, first) * (old / grown)[:, :, None, None]
    keep = (torch.arange(page, device=held.device)[None, :] < held[:, None])[:, None, :, None]
    as_bytes = pages.view(torch.uint8)
    as_bytes[first] = torch.where(keep, codes.to(pages.dtype).view(torch.uint8), as_bytes[first])
    scales[at] = fit[at]
    as_bytes[at, :, slot] = (x / fit[at][..., None]).to(pages.dtype).view(torch.uint8)


def _plain_attention(s):
    q, table, lengths = s["q"], s["page_table"], s["lengths"]
    tokens, heads, dim = q.shape
    seqs, kv_heads, most = table.shape[0], s["k_pages"].shape[1], s["most_new"]
    b, i = _sequence_of(s, tokens, seqs)
    rows = q.new_zeros((seqs, most, heads, dim), dtype=torch.float32)
    rows[b, i] = q.float()
    cu = s["cu_tokens"]
    new = torch.full((seqs,), most, device=q.device) if cu is None else cu[1:] - cu[:-1]

    def gather(pages, scales):
        at = table.clamp(min=0).long()
        x = _take(pages, at)
        if scales is not None:
            x *= scales[at][..., None, None]
        return x.transpose(1, 2).flatten(2, 3)                                   # [seqs, kv_heads, positions, dim]

    rows = rows.view(seqs, most, kv_heads, heads // kv_heads, dim).permute(0, 2, 1, 3, 4).flatten(2, 3)
    scores = rows @ gather(s["k_pages"], s["k_scales"]).transpose(-1, -2)
    scores *= s["scale"]
    seen = lengths[:, None] - new[:, None] + torch.arange(most, device=q.device)[None, :] + 1
    seen = torch.minimum(seen, lengths[:, None]).repeat_interleave(heads // kv_heads, dim=1)
    scores.masked_fill_((torch.arange(scores.shape[-1], device=q.device) >= seen[..., None])[:, None], -math.inf)
    top = scores.amax(dim=-1, keepdim=True)
    scores -= torch.where(top == -math.inf, 0.0, top)
    scores.exp_()
    total = scores.sum(dim=-1, keepdim=True)
    out = (scores @ gather(s["v_pages"], s["v_scales"])) / torch.where(total == 0, 1.0, total)
    out = out.view(seqs, kv_heads, most, heads // kv_heads, dim).permute(0, 2, 1, 3, 4).reshape(seqs, most, heads, dim)
    return out[b, i].bfloat16()


def work(case):
    new, start = _lengths(case)
    tokens, dim, heads, kv_heads = sum(new), case["dim"], case["heads"], case["kv_heads"]
    element = 2 if case["cache"] == BF16 else 1
    if case["op"] == "append":
        positions = len({p + i for n, p in zip(new, start) for i in range(n)})
        touched = sum((p + n - 1) // case["page"] - p // case["page"] + 1 for n, p in zip(new, start))
        moved = tokens * dim * (heads * 4 + 2 * kv_heads * (2 + element)) + positions * case["rot"] * 8
        return {"bytes": moved + (touched * kv_heads * 8 if element == 1 else 0), "flops": tokens * case["rot"] * (heads + kv_heads) * 3}
    pairs = cached = 0
    for b, (n, p) in enumerate(zip(new, start)):
        if b >= case["empty"]:
            pairs += n * p + n * (n + 1) // 2
            cached += n + p
    moved = tokens * heads * dim * 4 + cached * kv_heads * dim * 2 * element
    return {"bytes": moved + (-(-cached // case["page"]) * kv_heads * 8 if element == 1 else 0), "flops": 4 * dim * heads * pairs}


def exact(case, seed):
    s = prepare(case, seed)
    new, start = _lengths(case)
    at = 0
    if case["op"] == "attention":
        out = torch.zeros(s["q"].shape, dtype=torch.float64, device="cuda")
        group = case["heads"] // case["kv_heads"]
        for b, (n, length) in enumerate(zip(new, s["lengths"].tolist())):
            pages = s["page_table"][b, :-(-length // case["page"])].long()
            for h in range(case["kv_heads"] if length else 0):
                k, v = (x[pages, h].double() if c is None else x[pages, h].double() * c[pages, h].double()[:, None, None]
                        for x, c in ((s["k_pages"], s["k_scales"]), (s["v_pages"], s["v_scales"])))
                k, v = k.reshape(-1, case["dim"])[:length], v.reshape(-1, case["dim"])[:length]
                future = torch.arange(length, device="cuda")[None, :] > torch.arange(length - n, length, device="cuda")[:, None]
                for j in range(h * group, (h + 1) * group):
                    w = s["q"][at:at + n, j].double() @ k.T * s["scale"]
                    out[at:at + n, j] = torch.softmax(w.masked_fill(future, -math.inf), dim=-1) @ v
            at += n
        return out
    rot, dim = case["rot"], case["dim"]
    # a pair of elements as one complex number times the angle's
    first = torch.arange(rot // 2, device="cuda") * (1 if case["layout"] == "half" else 2)
    second = first + (rot // 2 if case["layout"] == "half" else 1)
    row_pos = torch.cat([torch.arange(p, p + n) for n, p in zip(new, start)]).cuda()
    turn = torch.complex(s["rope_cos"][row_pos][:, first].double(), s["rope_sin"][row_pos][:, first].double())[:, None]

    def rotated(x):
        y = x.double().clone()
        z = torch.complex(y[..., first], y[..., second]) * turn
        y[..., first], y[..., second] = z.real, z.imag
        return y

    result = {"q": rotated(s["q"])}
    for name, x in (("k", rotated(s["k"])), ("v", s["v"].double())):
        pages, scales = s[name + "_pages"].double(), s[name + "_scales"]
        scales = None if scales is None else scales.double().clone()
        at = 0
        for b, (n, p) in enumerate(zip(new, start)):
            for first_pos in range(p - p % case["page"], p + n, case["page"]):
                low, high = max(p, first_pos), min(p + n, first_pos + case["page"])
                to = int(s["page_table"][b, first_pos // case["page"]])
                rows, held = x[at + low - p:at + high - p].transpose(0, 1), low - first_pos
                if scales is not None:
                    old = scales[to].clone()
                    most = rows.abs().amax(dim=(1, 2)).float().double()
                    part, power = torch.frexp(most / E4M3_MAX)
                    need = torch.exp2((power - (part == 0.5).int()).clamp(*SCALE_EXPONENTS).double())
                    scales[to] = torch.maximum(old, need) if held else need
                    pages[to, :, :held] *= (old / scales[to])[:, None, None]
                    rows = rows / scales[to][:, None, None]
                pages[to, :, held:held + high - low] = rows
            at += n
        result[name + "_pages"], result[name + "_scales"] = pages, scales
    return result
