"""Cases of the serving operators of a decoder layer: the paged key/value cache (written, read back, attended to) and the
router of the experts.

Each case is one call as a serving program makes it. `run` computes it in its plain form, elementary torch operations in
32 bits (64 where 32 would lose what decides), or, with `own` set, through the framework. `exact` computes the
definitions in 64 bits.

The cache's memory is the layout that include/b200.h documents: arrays k, v (F16, or the int8 values of Q8_0) as
[page][kv_head][slot][dim], and for Q8_0 the scales k, v (F16) as [page][kv_head][slot][dim / 32], each array starting on
a multiple of 256 bytes.
"""

import importlib.util
import math
import os
import sys

import torch

own = False

_DEV = "cuda"
_pkg = None
_ctx = None


def _framework():
    """The package and one context of it (the package's folder name is not a Python identifier)."""
    global _pkg, _ctx
    if _pkg is None:
        name = "speechcpp_b200"
        if name not in sys.modules:
            root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
            folder = os.path.join(root, "speech.cpp_b200")
            spec = importlib.util.spec_from_file_location(name, os.path.join(folder, "__init__.py"), submodule_search_locations=[folder])
            module = importlib.util.module_from_spec(spec)
            sys.modules[name] = module
            spec.loader.exec_module(module)
        _pkg = sys.modules[name]
        _ctx = _pkg.Context(0)
    return _pkg, _ctx


# ---------------------------------------------------------------------------------------------------------------------
# cases
# ---------------------------------------------------------------------------------------------------------------------


def _attention(name, cache, seqs, tokens, max_len, heads, kv_heads, dim, page, lens):
    return dict(name=name, op="attention", cache=cache, seqs=seqs, tokens=tokens, max_len=max_len, heads=heads, kv_heads=kv_heads, dim=dim,
                page=page, lens=lens)


def _store(name, op, cache, seqs, tokens, max_len, kv_heads, dim, page, lens, out="f32"):
    return dict(name=name, op=op, cache=cache, seqs=seqs, tokens=tokens, max_len=max_len, kv_heads=kv_heads, dim=dim, page=page, lens=lens,
                out=out)


def _router(name, tokens, experts, top_k, score, bias, groups, keep, group_top, renorm, scale):
    return dict(name=name, op="router", tokens=tokens, experts=experts, top_k=top_k, score=score, bias=bias, groups=groups, keep=keep,
                group_top=group_top, renorm=renorm, scale=scale)


def listed():
    return [
        # one talker or ASR decoder step of one request: latency
        _attention("attend_step_f16", "f16", 1, 1, 517, 16, 8, 128, 16, "full"),
        # a batch of decoder steps at all lengths up to a few thousand positions
        _attention("attend_batch_f16", "f16", 64, 1, 4096, 16, 8, 128, 16, "ramp"),
        # the largest: a batch of long requests over a quantised cache
        _attention("attend_batch_q8_0", "q8_0", 32, 1, 16384, 16, 8, 128, 64, "ramp"),
        # one very long request, few key/value heads: the cache's length is what there is to split
        _attention("attend_long_q8_0", "q8_0", 1, 1, 131071, 32, 4, 128, 32, "full"),
        # a verify step: one token and four drafted ones of eight requests
        _attention("attend_verify_f16", "f16", 8, 5, 2050, 16, 8, 128, 32, "ramp"),
        # a padded batch with an empty and a one-token sequence, a group of five heads, pages of 48
        _attention("attend_ragged_q8_0", "q8_0", 7, 2, 777, 15, 3, 64, 48, "edges"),
        # a decode step's rows of 64 requests, quantised as they are written, and what the cache then holds of them
        _store("write_step_q8_0", "write", "q8_0", 64, 1, 600, 8, 128, 16, "ramp"),
        # a prompt of 1500 rows into an F16 cache
        _store("write_prompt_f16", "write", "f16", 1, 1500, 1500, 8, 128, 16, "full"),
        # the cached prefix of one request as F16, for attention over a prompt's block
        _store("read_prefix_f16", "read", "q8_0", 1, 1031, 1031, 8, 128, 32, "full", "f16"),
        # the caches of a batch taken out as values
        _store("read_batch_f32", "read", "q8_0", 24, 4001, 5000, 8, 128, 64, "ramp", "f32"),
        # one step of one request, and of a batch: softmax scores, the eight best of 128, weights renormalised
        _router("route_step", 1, 128, 8, "softmax", False, 1, 1, 1, True, 1.0),
        # a prompt's rows: sigmoid scores, a balance bias, four groups of eight kept
        _router("route_prompt_groups", 16384, 256, 8, "sigmoid", True, 8, 4, 2, True, 2.5),
    ]


def _spread(rng, low, high):
    """A whole number whose logarithm is spread evenly over [low, high]."""
    if high <= low:
        return low
    return max(low, min(high, int(round(math.exp(rng.uniform(math.log(low), math.log(high + 0.49)))))))


def draw(rng):
    kind = rng.choice(["attention", "attention", "write", "read", "router"])
    if kind == "router":
        experts = rng.choice([8, 60, 64, 128, 160, 256, 384])
        groups = rng.choice([1, 1, 2, 4])
        keep = rng.randint(1, groups)
        top_k = rng.randint(1, min(16, experts // groups * keep))
        score = rng.choice(["softmax", "sigmoid"])
        bias = rng.choice([True, False])
        return _drawn(_router("", _spread(rng, 1, 12000), experts, top_k, score, bias, groups, keep, rng.choice([1, 2]), rng.choice([True, False]),
                              rng.choice([1.0, 2.5])))
    kv_heads = rng.choice([1, 2, 3, 4, 8])
    dim = rng.choice([64, 96, 128, 128, 256])
    cache = rng.choice(["f16", "q8_0"])
    page = rng.choice([16, 32, 48, 64, 128])
    lens = rng.choice(["full", "ramp", "edges"])
    if kind == "attention":
        seqs = _spread(rng, 1, 96)
        tokens = rng.choice([1, 1, 1, 2, 3, 5, 8])
        max_len = _spread(rng, tokens, min(100000, (1 << 27) // (seqs * kv_heads * dim)))
        return _drawn(_attention("", cache, seqs, tokens, max_len, kv_heads * rng.choice([1, 2, 3, 4, 8]), kv_heads, dim, page, lens))
    tokens = _spread(rng, 1, 4000)
    seqs = _spread(rng, 1, max(1, min(64, (1 << 25) // (tokens * kv_heads * dim))))
    max_len = tokens + rng.randint(0, tokens)
    return _drawn(_store("", kind, cache, seqs, tokens, max_len, kv_heads, dim, page, lens, rng.choice(["f32", "f16"])))


def _drawn(case):
    del case["name"]
    return case


def _lens(case):
    """The sequences' lengths (a case's own; the seed only says whose they are)."""
    n, top = case["seqs"], case["max_len"]
    if case["lens"] == "full":
        return [top] * n
    got = [max(1, top - (top * 7 // 8) * i // n) for i in range(n)]
    if case["lens"] == "edges":  # nothing, one token, one page exactly, one token past a page
        for i, v in zip(range(n - 1, 0, -1), (0, 1, case["page"], case["page"] + 1)):
            got[i] = min(v, top)
    return got


def _starts(case, lens):
    """The first position read of each sequence."""
    return [max(0, v - case["tokens"]) for v in lens]


# ---------------------------------------------------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------------------------------------------------


def _arrays(case, pages):
    """(offset, shape, type) of each array of the cache, and the bytes of all."""
    rows = [pages, case["kv_heads"], case["page"]]
    q8 = case["cache"] == "q8_0"
    value, size = (torch.int8, 1) if q8 else (torch.float16, 2)
    kinds = [(rows + [case["dim"]], value, size)] * 2 + ([(rows + [case["dim"] // 32], torch.float16, 2)] * 2 if q8 else [])
    got, at = [], 0
    for shape, kind, size in kinds:
        got.append((at, shape, kind))
        at += -(-math.prod(shape) * size // 256) * 256
    return got, at


def _views(case, memory, pages):
    out = []
    for at, shape, kind in _arrays(case, pages)[0]:
        size = 1 if kind == torch.int8 else 2
        out.append(memory[at : at + math.prod(shape) * size].view(kind).view(shape))
    return out


def _quantise(x):
    """x [..., dim] in 32 bits to Q8_0: int8 values, F16 scales. Each quotient and product is rounded to 32 bits once."""
    b = x.unflatten(-1, (-1, 32))
    d = (b.abs().amax(-1).double() / 127.0).float()
    inv = torch.where(d != 0, (1.0 / d.double()).float(), torch.zeros_like(d))
    q = (b * inv[..., None]).double()
    q = torch.sign(q) * torch.floor(q.abs() + 0.5)
    return q.to(torch.int8).flatten(-2), d.half()


def _values(q, d):
    """What Q8_0 stands for: the scale times the whole number, exact in 32 bits."""
    return (q.float().unflatten(-1, (-1, 32)) * d.float()[..., None]).flatten(-2)


def _rows(shape, gen, outliers):
    """Rows of a key or value projection: normal values, some channels larger than the others."""
    x = torch.randn(shape, generator=gen, device=_DEV)
    return x * (1.0 + outliers * (torch.arange(shape[-1], device=_DEV) % 37 == 5))


def prepare(case, seed):
    gen = torch.Generator(device=_DEV)
    gen.manual_seed(seed)
    s = dict(case=case)
    if case["op"] == "router":
        s["logits"] = torch.randn(case["tokens"], case["experts"], generator=gen, device=_DEV) * 1.5
        s["bias"] = torch.randn(case["experts"], generator=gen, device=_DEV) * 0.05 if case["bias"] else None
        if own:
            _framework()
        return s
    lens = torch.tensor(_lens(case), dtype=torch.int32, device=_DEV)
    lens = lens[torch.randperm(case["seqs"], generator=gen, device=_DEV)]
    width = -(-case["max_len"] // case["page"])
    pages = case["seqs"] * width
    table = torch.randperm(pages, generator=gen, device=_DEV).view(case["seqs"], width).to(torch.int32)
    memory = torch.zeros(_arrays(case, pages)[1], dtype=torch.uint8, device=_DEV)
    views = _views(case, memory, pages)
    s.update(lens=lens, table=table, memory=memory, views=views)
    if case["op"] != "write":  # a cache that sequences have filled
        for which, outliers in ((0, 4.0), (1, 0.0)):
            for a in range(0, pages, 1024):
                x = _rows(list(views[which][a : a + 1024].shape), gen, outliers)
                if case["cache"] == "q8_0":
                    views[which][a : a + 1024], views[2 + which][a : a + 1024] = _quantise(x)
                else:
                    views[which][a : a + 1024] = x
    rows = [case["seqs"], case["tokens"]]
    if case["op"] == "attention":
        s["q"] = torch.randn(rows + [case["heads"], case["dim"]], generator=gen, device=_DEV) * 1.7
        s["scale"] = 1.0 / math.sqrt(case["dim"])
    else:
        s["start"] = (lens - case["tokens"]).clamp(min=0) if case["op"] == "write" or case["max_len"] > case["tokens"] else None
        kind = torch.float16 if case["out"] == "f16" else torch.float32
        shape = rows + [case["kv_heads"], case["dim"]]
        if case["op"] == "write":
            s["k"], s["v"] = _rows(shape, gen, 4.0), _rows(shape, gen, 0.0)
        if case["op"] == "read" or case["cache"] == "q8_0":
            s["k_out"], s["v_out"] = (torch.zeros(shape, dtype=kind, device=_DEV) for _ in range(2))
    if own:
        pkg, ctx = _framework()
        qtype = pkg.Q8_0 if case["cache"] == "q8_0" else pkg.F16
        s["cache"] = ctx.kv_cache(qtype, case["kv_heads"], case["dim"], case["page"], pages, data=memory)  # the program's handle
    return s


# ---------------------------------------------------------------------------------------------------------------------
# one pass
# ---------------------------------------------------------------------------------------------------------------------


def run(s):
    return _run_own(s) if own else _run_plain(s)


def _run_own(s):
    case = s["case"]
    ctx = _ctx
    if case["op"] == "router":
        return ctx.moe_router(s["logits"], case["top_k"], bias=s["bias"], score=case["score"], n_group=case["groups"], topk_group=case["keep"],
                              group_top=case["group_top"], renorm=case["renorm"], scale=case["scale"])
    if case["op"] == "attention":
        return ctx.kv_attention(s["cache"], s["q"], s["table"], s["lens"], s["scale"])
    if case["op"] == "write":
        ctx.kv_write(s["cache"], s["k"], s["v"], s["table"], s["lens"])
        if case["cache"] == "f16":
            return s["views"]
    return ctx.kv_read(s["cache"], s["table"], s["lens"], start=s["start"], k=s["k_out"], v=s["v_out"])


def _run_plain(s):
    return {"router": _plain_router, "attention": _plain_attention, "write": _plain_write, "read": _plain_read}[s["case"]["op"]](s)


def _gathered(s, which):
    """The sequences' cached rows as [seq][kv_head][position][dim] in 32 bits."""
    table = s["table"].long()
    x = s["views"][which][table]
    x = _values(x, s["views"][2 + which][table]) if s["case"]["cache"] == "q8_0" else x.float()
    return x.transpose(1, 2).flatten(2, 3)


def _plain_attention(s):
    case = s["case"]
    n, groups = case["tokens"], case["heads"] // case["kv_heads"]
    k = _gathered(s, 0)
    q = s["q"].unflatten(2, (case["kv_heads"], groups)).permute(0, 2, 1, 3, 4).flatten(2, 3)  # [seq][kv_head][token, group][dim]
    score = torch.matmul(q, k.transpose(-1, -2)) * s["scale"]
    del k
    seen = s["lens"].long()[:, None] - n + 1 + torch.arange(n, device=_DEV)[None, :]
    seen = seen.repeat_interleave(groups, 1)[:, None, :, None]
    score = torch.where(torch.arange(score.shape[-1], device=_DEV) < seen, score, torch.full_like(score, -math.inf))
    top = score.amax(-1, keepdim=True)
    weight = torch.exp(score - torch.where(top > -math.inf, top, torch.zeros_like(top)))
    total = weight.sum(-1, keepdim=True)
    v = _gathered(s, 1)
    v = torch.where(torch.arange(v.shape[2], device=_DEV)[:, None] < s["lens"].long()[:, None, None, None], v, torch.zeros_like(v))
    out = torch.matmul(weight, v)
    out = torch.where(total > 0, out / total, torch.zeros_like(out))
    return out.unflatten(2, (n, groups)).permute(0, 2, 1, 3, 4).flatten(2, 3).contiguous()


def _places(s, first):
    """(page, slot, whether there is such a row) of `tokens` positions from `first` [seq]."""
    case = s["case"]
    at = first.long()[:, None] + torch.arange(case["tokens"], device=_DEV)[None, :]
    there = (at >= 0) & (at < s["lens"].long()[:, None])
    at = at.clamp(0, s["table"].shape[1] * case["page"] - 1)
    return s["table"].long().gather(1, at // case["page"]), at % case["page"], there


def _plain_write(s):
    case = s["case"]
    page, slot, there = _places(s, s["lens"] - case["tokens"])
    page, slot = page[there], slot[there]
    for which, x in ((0, s["k"]), (1, s["v"])):
        x = x[there]
        if case["cache"] == "q8_0":
            q, d = _quantise(x)
            s["views"][which][page, :, slot] = q
            s["views"][2 + which][page, :, slot] = d
        else:
            s["views"][which][page, :, slot] = x.half()
    return _plain_read(s) if case["cache"] == "q8_0" else s["views"]


def _plain_read(s):
    first = s["start"] if s["start"] is not None else torch.zeros_like(s["lens"])
    page, slot, there = _places(s, first)
    out = []
    for which, to in ((0, s["k_out"]), (1, s["v_out"])):
        x = s["views"][which][page, :, slot]
        x = _values(x, s["views"][2 + which][page, :, slot]) if s["case"]["cache"] == "q8_0" else x.float()
        out.append(torch.where(there[..., None, None], x.to(to.dtype), to))
    return tuple(out)


def _scores(logits, score):
    """Softmax or sigmoid of each row in 64 bits, as scores of the experts are ordered by their last bits."""
    x = logits.double()
    if score == "sigmoid":
        return 1.0 / (1.0 + torch.exp(-x))
    e = torch.exp(x - x.amax(-1, keepdim=True))
    return e / e.sum(-1, keepdim=True)


def _plain_router(s):
    case = s["case"]
    p = _scores(s["logits"], case["score"])
    choice = p + s["bias"].double() if case["bias"] else p
    if case["groups"] > 1:
        best = choice.unflatten(-1, (case["groups"], -1))
        best = best.topk(min(case["group_top"], best.shape[-1]), -1).values.sum(-1)
        kept = torch.sort(best, dim=-1, descending=True, stable=True).indices[:, : case["keep"]]
        stays = torch.zeros_like(best).scatter_(-1, kept, 1.0).repeat_interleave(case["experts"] // case["groups"], -1)
        choice = torch.where(stays > 0, choice, torch.full_like(choice, -math.inf))
    ids = torch.sort(choice, dim=-1, descending=True, stable=True).indices[:, : case["top_k"]]
    w = p.gather(-1, ids)
    if case["renorm"]:
        w = w / w.sum(-1, keepdim=True)
    return ids.to(torch.int32), (w * case["scale"]).float()


# ---------------------------------------------------------------------------------------------------------------------
# what a pass cannot do without
# ---------------------------------------------------------------------------------------------------------------------


def work(case):
    if case["op"] == "router":
        t = case["tokens"]
        return {"bytes": 4 * t * case["experts"] + 8 * t * case["top_k"], "flops": 4 * t * case["experts"]}
    lens = _lens(case)
    row = case["kv_heads"] * case["dim"]
    cached = 2 * row * (34 / 32 if case["cache"] == "q8_0" else 2)  # bytes of one position
    if case["op"] == "attention":
        n = case["tokens"]
        seen = sum(max(0, v - n + 1 + r) for v in lens for r in range(n))
        return {"bytes": cached * sum(lens) + 8 * case["seqs"] * n * case["heads"] * case["dim"], "flops": 4 * case["heads"] * case["dim"] * seen}
    moved = sum(v - a for v, a in zip(lens, _starts(case, lens))) if case["op"] == "write" or case["max_len"] > case["tokens"] else sum(lens)
    out = 2 * row * (2 if case["out"] == "f16" else 4)
    if case["op"] == "read":
        return {"bytes": moved * (cached + out), "flops": 2 * moved * row}
    again = cached + out if case["cache"] == "q8_0" else 0  # the rows taken out again
    return {"bytes": moved * (8 * row + cached + again), "flops": 8 * moved * row}


# ---------------------------------------------------------------------------------------------------------------------
# the definitions in 64 bits
# ---------------------------------------------------------------------------------------------------------------------


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "router":
        return None, _exact_weights(s)
    if case["op"] == "attention":
        return _exact_attention(s)
    if case["op"] == "write" and case["cache"] == "f16":
        return _exact_cache(s)
    return _exact_rows(s)


def _stored(s, which, i, kv_head, first, last):
    """Positions [first, last) of sequence i as the cache holds them, in 64 bits."""
    case, table = s["case"], s["table"][i].tolist()
    width = case["page"]
    got = []
    for b in range(first // width, -(-last // width)):
        rows = slice(max(first - b * width, 0), min(last - b * width, width))
        x = s["views"][which][table[b], kv_head, rows].double()
        if case["cache"] == "q8_0":
            x = x * s["views"][2 + which][table[b], kv_head, rows].double().repeat_interleave(32, -1)
        got.append(x)
    return torch.cat(got, -2)


def _exact_attention(s):
    case = s["case"]
    out = torch.zeros(s["q"].shape, dtype=torch.float64, device=_DEV)
    groups, lens = case["heads"] // case["kv_heads"], s["lens"].tolist()
    for i, size in enumerate(lens):
        if size == 0:
            continue
        every = slice(0, case["kv_heads"])
        k, v = _stored(s, 0, i, every, 0, size), _stored(s, 1, i, every, 0, size)
        for r in range(case["tokens"]):
            seen = size - case["tokens"] + r + 1
            if seen <= 0:
                continue
            q = s["q"][i, r].double().view(case["kv_heads"], groups, case["dim"])
            w = torch.softmax(torch.einsum("hgd,htd->hgt", q, k[:, :seen]) * s["scale"], -1)
            out[i, r] = torch.einsum("hgt,htd->hgd", w, v[:, :seen]).reshape(case["heads"], case["dim"])
    return out


def _exact_rows(s):
    case = s["case"]
    lens = s["lens"].tolist()
    out = [torch.zeros(s["k_out"].shape, dtype=torch.float64, device=_DEV) for _ in range(2)]
    for i, size in enumerate(lens):
        first = 0 if s["start"] is None else int(s["start"][i])
        last = min(size, first + case["tokens"])
        if last <= first:
            continue
        for which in range(2):
            if case["op"] == "read":
                got = _stored(s, which, i, slice(0, case["kv_heads"]), first, last).transpose(0, 1)
            else:
                rows = (s["k"], s["v"])[which][i, case["tokens"] - (last - first) :]
                blocks = rows.double().reshape(-1, 32)
                scale = (blocks.abs().max(1).values / 127.0).float()  # the definition's own roundings: the scale, its
                inverse = torch.zeros_like(scale)                     # inverse, the product, and the scale as stored
                inverse[scale > 0] = (1.0 / scale[scale > 0].double()).float()
                product = (blocks * inverse.double()[:, None]).float().double()
                whole = torch.where(product < 0, torch.ceil(product - 0.5), torch.floor(product + 0.5))
                got = (whole * scale.half().double()[:, None]).reshape(rows.shape)
            out[which][i, : last - first] = got
    return tuple(out)


def _exact_cache(s):
    """The whole F16 cache after the rows are written, each row's values as they came."""
    case, table = s["case"], s["table"].tolist()
    out = [x.double() for x in s["views"]]
    for i, size in enumerate(s["lens"].tolist()):
        first, width = max(0, size - case["tokens"]), case["page"]
        for which, rows in enumerate((s["k"][i].double(), s["v"][i].double())):
            for b in range(first // width, -(-size // width)):
                at, to = max(first, b * width), min(size, (b + 1) * width)
                r = at - (size - case["tokens"])
                out[which][table[i][b], :, at - b * width : to - b * width] = rows[r : r + to - at].transpose(0, 1)
    return out


def _exact_weights(s):
    """The chosen experts' weights: the choice is made again here, one group and one expert at a time."""
    case = s["case"]
    x = s["logits"].double()
    p = torch.sigmoid(x) if case["score"] == "sigmoid" else torch.softmax(x, -1)
    choice = p + (s["bias"].double() if case["bias"] else 0.0)
    size = case["experts"] // case["groups"]
    if case["groups"] > 1:
        parts = choice.view(-1, case["groups"], size)
        first = parts.max(-1)
        best = first.values
        if case["group_top"] == 2 and size > 1:
            best = best + parts.scatter(-1, first.indices[..., None], -math.inf).max(-1).values
        open_ = torch.zeros_like(parts, dtype=torch.bool)
        for _ in range(case["keep"]):
            g = best.argmax(-1, keepdim=True)
            open_.scatter_(1, g[..., None].expand(-1, -1, size), True)
            best = best.scatter(-1, g, -math.inf)
        choice = choice.masked_fill(~open_.view(choice.shape), -math.inf)
    got = []
    for _ in range(case["top_k"]):
        e = choice.argmax(-1, keepdim=True)
        got.append(p.gather(-1, e))
        choice = choice.scatter(-1, e, -math.inf)
    w = torch.cat(got, -1)
    return (w / w.sum(-1, keepdim=True) if case["renorm"] else w) * case["scale"]
