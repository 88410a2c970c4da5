"""The timed work of a paged KV cache in 8 bits, and of requests that share a prefix (mongoose_amd.engine, HIPPaged):

  store      rotary positions, K and V rows quantized into their slots (int8, a scale a KV head's row), and the same rows read back
             as fp32                                                                    HIPPaged.Store, HIPPaged.Load
  load       the last positions of every request, or all of them, out of the pages as fp32 rows           HIPPaged.Load
  attention  new tokens of every request (one or many) over the request's pages of an 8-bit cache          HIPPaged.Attention
  shared     the same for groups of requests whose first positions lie in the same pages, any cache format
                                                                                        HIPPaged.PlanShared, HIPPaged.Attention

`own` false: the same in elementary torch operations, 32 bits (64 for the turned K rows, whose rounding to 8 bits is at stake), the
requests of a batch padded to the longest.  Lengths come from the case, values from the seed.
"""
import math
import random

import torch

own = False

_SHAPES = ((32, 8, 128), (32, 4, 64), (14, 2, 64), (8, 8, 64))       # heads, KV heads, head size of the benchmark configurations
_FORMATS = {"f32": 0, "f16": 1, "q8": 8}
_MOST = 2048 * 32 * 12000                                            # scores of the largest attention, padded


# ---------------------------------------------------------------------------------------------------------------------
# cases
# ---------------------------------------------------------------------------------------------------------------------
def _case(op, heads, kvheads, hd, fmt, page, reqs, new, cached, singles=0.0, cap=0.0, slopes=False, groups=0, prefix=(0, 0)):
    return {"op": op, "heads": heads, "kvheads": kvheads, "hd": hd, "fmt": fmt, "page": page, "reqs": reqs, "new_lo": new[0],
            "new_hi": new[1], "cached_lo": cached[0], "cached_hi": cached[1], "singles": singles, "cap": cap, "slopes": slopes,
            "groups": groups, "prefix_lo": prefix[0], "prefix_hi": prefix[1]}


def listed():
    return [
        # the rows of a decode step of the 0.5B shape
        dict(_case("store", 14, 2, 64, "q8", 16, 48, (1, 1), (0, 3000)), name="store-tokens"),
        # chunks of three prompts of the 8B shape that arrive together
        dict(_case("store", 32, 8, 128, "q8", 64, 3, (900, 1700), (0, 500)), name="store-chunks"),
        # the last rows of a few requests, to be looked at on the host
        dict(_case("load", 14, 2, 64, "q8", 16, 7, (1, 60), (10, 900)), name="load-tails"),
        # two conversations that leave the card whole, 8B shape
        dict(_case("load", 32, 8, 128, "q8", 64, 2, (9000, 21000), (0, 0)), name="load-contexts"),
        # one user, a short conversation: all latency
        dict(_case("attention", 14, 2, 64, "q8", 16, 1, (1, 1), (500, 500)), name="token-short"),
        # a decode step of a busy server, conversations of very different lengths, 8B shape
        dict(_case("attention", 32, 8, 128, "q8", 16, 48, (1, 1), (100, 8000)), name="token-batch"),
        # one user with a book in the cache
        dict(_case("attention", 32, 8, 128, "q8", 64, 1, (1, 1), (120001, 120001)), name="token-long"),
        # a chunk of a long prompt: the matrix cores' case
        dict(_case("attention", 32, 8, 128, "q8", 64, 1, (2048, 2048), (9700, 9700)), name="chunk"),
        # a few drafted tokens a request, capped scores
        dict(_case("attention", 32, 4, 64, "q8", 32, 24, (3, 7), (300, 4000), cap=50.0), name="drafts-capped"),
        # eight answers to one question, toy shape, the default cache format, a bias by distance: all latency
        dict(_case("shared", 8, 8, 64, "f32", 16, 8, (1, 1), (0, 60), slopes=True, groups=1, prefix=(700, 700)), name="shared-answers"),
        # a decode step of 64 requests behind one long system prompt, 8B shape
        dict(_case("shared", 32, 8, 128, "f16", 16, 64, (1, 1), (30, 900), groups=1, prefix=(8001, 8001)), name="shared-system"),
        # four prompts of different lengths, some tens of requests behind them, some with a turn of several rows; 8 bits
        dict(_case("shared", 32, 8, 128, "q8", 32, 80, (1, 40), (0, 700), singles=0.8, groups=4, prefix=(900, 6000)), name="shared-groups"),
    ]


def _between(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(("store", "load", "attention", "attention", "shared", "shared"))
    page = rng.choice((8, 16, 32, 64, 128))
    heads, kvheads, hd = rng.choice(_SHAPES)
    if op == "store":
        reqs = _between(rng, 1, 64)
        new = max(1, _between(rng, 1, 4096) // reqs)
        return _case(op, heads, kvheads, hd, "q8", page, reqs, (rng.choice((1, new)), new), (0, rng.choice((0, 100, 2000))))
    if op == "load":
        reqs = _between(rng, 1, 64)
        rows = max(1, _between(rng, 1, 30000) // reqs)
        return _case(op, heads, kvheads, hd, rng.choice(("q8", "q8", "f16", "f32")), page, reqs, (rng.choice((1, rows)), rows), (0, rng.choice((0, 0, 700))))
    cap, slopes = rng.choice(((0.0, False), (0.0, False), (30.0, False), (0.0, True)))
    while True:
        reqs, new = _between(rng, 1, 64), rng.choice((1, 1, _between(rng, 2, 2048 if op == "attention" else 200)))
        cached, prefix = _between(rng, 1, 60000 if op == "attention" else 2000), _between(rng, 20, 12000) if op == "shared" else 0
        if reqs * heads * new * (cached + prefix + new) <= _MOST and reqs * (cached + prefix + new) <= 400000:
            break
    fmt = "q8" if op == "attention" else rng.choice(("q8", "f16", "f32"))
    return _case(op, heads, kvheads, hd, fmt, page, reqs, (rng.choice((1, new)), new), (rng.choice((0, cached // 2, cached)), cached), singles=rng.choice((0.0, 0.5)),
                 cap=cap, slopes=slopes, groups=rng.randint(1, max(1, reqs // 3)) if op == "shared" else 0, prefix=(rng.choice((prefix, prefix // 3)), prefix))


def _sizes(case):
    """What the case fixes of its batch: new and cached tokens of every request -- the latter with its group's prefix --, the first
    request of every group (and the end), the groups' prefixes; the same for every seed."""
    rng = random.Random(repr(sorted((k, v) for k, v in case.items() if k != "name")))
    n, groups = case["reqs"], case["groups"]
    first = [0] + sorted(rng.sample(range(1, n), groups - 1)) + [n] if groups else [0]
    prefix = [rng.randint(case["prefix_lo"], case["prefix_hi"]) for _ in range(groups)]
    new, cached = [], []
    for r in range(n):
        new.append(1 if rng.random() < case["singles"] else rng.randint(case["new_lo"], case["new_hi"]))
        cached.append(rng.randint(case["cached_lo"], case["cached_hi"]) + sum(p for g, p in enumerate(prefix) if first[g] <= r < first[g + 1]))
    return new, cached, first, prefix


def _row_bytes(case):
    """A position's K (or V) row in the cache."""
    width = case["kvheads"] * case["hd"]
    return {"f32": 4 * width, "f16": 2 * width, "q8": width + 4 * case["kvheads"]}[case["fmt"]]


def work(case):
    h, kv, hd = case["heads"], case["kvheads"], case["hd"]
    new, cached, first, prefix = _sizes(case)
    rows, row = sum(new), _row_bytes(case)
    if case["op"] == "store":
        return {"bytes": rows * (2 * h * hd * 4 + 2 * kv * hd * (4 + 4) + 2 * row + hd * 4 + 8), "flops": rows * (3 * h + 9 * kv) * hd}
    if case["op"] == "load":
        return {"bytes": rows * 2 * (row + kv * hd * 4), "flops": rows * 2 * kv * hd}
    positions = sum(n + c for n, c in zip(new, cached)) - sum(p * (first[g + 1] - first[g] - 1) for g, p in enumerate(prefix))
    return {"bytes": 2 * rows * h * hd * 4 + 2 * positions * row, "flops": 4 * hd * h * sum(n * c + n * (n + 1) // 2 for n, c in zip(new, cached))}


# ---------------------------------------------------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------------------------------------------------
def _ints(values, dev):
    return torch.tensor(values, dtype=torch.int32, device=dev)


def _done(rc):
    if rc:
        from mongoose_amd import engine as E
        raise RuntimeError(E.last_error())


def _stream():
    return torch.cuda.current_stream().cuda_stream


def _pool(case, pages, g, dev, channel):
    """A pool of the cache's format with rows in all its pages: normal values, channels of the given sizes."""
    kv, hd, page = case["kvheads"], case["hd"], case["page"]
    kind = torch.float16 if case["fmt"] == "f16" else torch.float32
    x = torch.randn((pages, page, kv, hd), generator=g, device=dev, dtype=kind).mul_(channel.to(kind))
    if case["fmt"] != "q8":
        return x.reshape(pages, page, kv * hd)
    scale = x.abs().amax(-1) / 127
    q = torch.round(x / scale[..., None]).to(torch.int8)
    # int8 [pages, page, kv * hd], then the scales [pages, kv, page]
    return torch.cat((q.reshape(-1).view(torch.uint8), scale.transpose(1, 2).contiguous().reshape(-1).view(torch.uint8)))


def _parts(case, pool, pages):
    """(int8 rows, scales) of an 8-bit pool."""
    kv, hd, page = case["kvheads"], case["hd"], case["page"]
    n = pages * page * kv * hd
    return pool[:n].view(torch.int8).view(pages, page, kv, hd), pool[n:].view(torch.float32).view(pages, kv, page)


def prepare(case, seed):
    dev = torch.device("cuda")
    g = torch.Generator(device=dev)
    g.manual_seed(seed)
    new, cached, first, prefix = _sizes(case)
    reqs, page, h, kv, hd = case["reqs"], case["page"], case["heads"], case["kvheads"], case["hd"]
    lens = [n + c for n, c in zip(new, cached)]
    rows, width = sum(new), -(-max(lens) // page) + 1
    # pages of a request's own, behind those that lie wholly in its group's prefix
    common = [0] * reqs
    for k, p in enumerate(prefix):
        common[first[k]:first[k + 1]] = [p // page] * (first[k + 1] - first[k])
    mine = [-(-n // page) - c for n, c in zip(lens, common)]
    theirs = [p // page for p in prefix]
    used = sum(mine) + sum(theirs)
    pages = used + used // 8 + 1                                         # a pool that is nearly full, in the order of its use
    order = torch.randperm(pages, generator=g, device=dev)[:used].to(torch.int32)
    at = torch.arange(width, device=dev)
    count, before = torch.tensor(mine, device=dev), torch.tensor(common, device=dev)
    start = torch.cumsum(count, 0) - count
    entry = start[:, None] + at - before[:, None]
    group0 = torch.tensor([sum(mine) + sum(theirs[:k]) for k in range(len(prefix)) for _ in range(first[k + 1] - first[k])] or [0] * reqs, device=dev)
    entry = torch.where(at < before[:, None], group0[:, None] + at, entry)
    held = at < (before + count)[:, None]
    s = {"case": case, "rows": rows, "pages": pages, "newMost": max(new), "lenMost": max(lens),
         "table": torch.where(held, order[entry.clamp(0, used - 1)], 0).to(torch.int32).contiguous(),
         "rowStart": _ints([sum(new[:r]) for r in range(reqs + 1)], dev), "lens": _ints(lens, dev),
         "groupStart": _ints(first, dev), "sharedLens": _ints(prefix, dev),
         "request": torch.repeat_interleave(torch.arange(reqs, device=dev), torch.tensor(new, device=dev))}
    if case["groups"]:
        # the rest of a prefix that ends inside a page: each request has a copy of the group's first one's rows
        s["copies"] = [(first[k], r, p) for k, p in enumerate(prefix) if p % page for r in range(first[k] + 1, first[k + 1])]
    channel = torch.exp(0.4 * torch.randn((kv, hd), generator=g, device=dev))             # channels of K differ in size, as trained ones do
    s["K"] = _pool(case, pages, g, dev, channel)
    s["V"] = _pool(case, pages, g, dev, torch.ones_like(channel))
    if case["groups"]:
        _copy_ends(s)
    if case["op"] == "store":
        qkv = torch.randn((rows, (h + 2 * kv) * hd), generator=g, device=dev)             # rows of one projection
        s["q"], s["k"], s["v"] = qkv[:, :h * hd], qkv[:, h * hd:(h + kv) * hd], qkv[:, (h + kv) * hd:]
        s["positions"] = (torch.cat([torch.arange(c, n, device=dev) for c, n in zip(cached, lens)])).to(torch.int32)
        place = s["positions"].long()
        s["slots"] = (s["table"][s["request"], place // page].long() * page + place % page).to(torch.int32)
        far = max(lens)
        angle = torch.arange(far, device=dev, dtype=torch.float64)[:, None] * 5e5 ** (-torch.arange(hd // 2, device=dev, dtype=torch.float64) * 2 / hd)
        s["cos"], s["sin"], s["far"] = torch.cos(angle).float(), torch.sin(angle).float(), far
    elif case["op"] != "load":
        s["q"] = 1.5 * torch.randn((rows, h * hd), generator=g, device=dev)
        s["slopes"] = torch.exp2(-8.0 * torch.arange(1, h + 1, device=dev) / h) if case["slopes"] else None
    if own:
        from mongoose_amd import engine as E
        p = s["paged"] = E.NewHIPPaged(E.NewHIP(), h, kv, hd, page, pages, _FORMATS[case["fmt"]], reqs, rows, width * page)
        if p is None:
            raise RuntimeError(E.last_error())
        if case["op"] in ("store", "load"):
            s["kOut"], s["vOut"] = (torch.empty((rows, kv * hd), device=dev) for _ in range(2))
        if case["op"] != "load":
            s["out"] = torch.empty((rows, h * hd), device=dev)
        if case["op"] == "attention":
            _done(p.Plan(s["rowStart"].data_ptr(), s["lens"].data_ptr(), reqs, rows, 0, None, _stream()))
        if case["op"] == "shared":
            _done(p.Share())
            _done(p.PlanShared(s["rowStart"].data_ptr(), s["lens"].data_ptr(), reqs, rows, s["newMost"], s["groupStart"].data_ptr(), s["sharedLens"].data_ptr(),
                               case["groups"], _stream()))
    return s


def _copy_ends(s):
    page = s["case"]["page"]
    if not s["copies"]:
        return
    a, b, p = (torch.tensor(x, device=s["table"].device) for x in zip(*s["copies"]))
    source, target = s["table"][a, p // page].long(), s["table"][b, p // page].long()
    keep = torch.arange(page, device=p.device) < (p % page)[:, None]
    for name in ("K", "V"):
        if s["case"]["fmt"] != "q8":
            x = s[name]
            x[target] = torch.where(keep[..., None], x[source], x[target])
        else:
            q, scale = _parts(s["case"], s[name], s["pages"])
            q[target] = torch.where(keep[..., None, None], q[source], q[target])
            scale[target] = torch.where(keep[:, None], scale[source], scale[target])


# ---------------------------------------------------------------------------------------------------------------------
# one pass
# ---------------------------------------------------------------------------------------------------------------------
def run(s):
    return {"store": _store, "load": _load, "attention": _attend, "shared": _attend}[s["case"]["op"]](s)


def _load_own(s, stream):
    kOut, vOut = s["kOut"], s["vOut"]
    _done(s["paged"].Load(s["K"].data_ptr(), s["V"].data_ptr(), s["table"].data_ptr(), s["rowStart"].data_ptr(), s["lens"].data_ptr(), s["case"]["reqs"], s["rows"],
                          kOut.data_ptr(), kOut.stride(0), vOut.data_ptr(), vOut.stride(0), stream))


def _store(s):
    c = s["case"]
    if own:
        st, q, k, v, out = _stream(), s["q"], s["k"], s["v"], s["out"]
        _done(s["paged"].Store(q.data_ptr(), k.data_ptr(), v.data_ptr(), q.stride(0), k.stride(0), v.stride(0), out.data_ptr(), out.stride(0), s["K"].data_ptr(),
                               s["V"].data_ptr(), s["slots"].data_ptr(), s["positions"].data_ptr(), s["rows"], s["cos"].data_ptr(), s["sin"].data_ptr(), s["far"], st))
        _load_own(s, st)
        return {"q": out, "k": s["kOut"], "v": s["vOut"]}
    hd, kv, page, at = c["hd"], c["kvheads"], c["page"], s["positions"].long()
    cos, sin = s["cos"][at][:, None, :], s["sin"][at][:, None, :]

    def turned(x, cos, sin):
        a, b = x.reshape(s["rows"], -1, 2, hd // 2).unbind(2)
        return torch.stack((a * cos - b * sin, a * sin + b * cos), 2).reshape(s["rows"], -1)

    slot = s["slots"].long()
    out = {"q": turned(s["q"], cos, sin)}
    for name, pool, x in (("k", "K", turned(s["k"].double(), cos.double(), sin.double()).float()), ("v", "V", s["v"])):
        rows, scales = _parts(c, s[pool], s["pages"])
        x = x.reshape(s["rows"], kv, hd)
        scale = (x.abs().amax(-1).double() / 127).float()
        size = torch.floor(x.double().abs() / scale.double()[..., None] + 0.5)           # half away from zero
        rows.view(-1, kv, hd)[slot] = (size * torch.sign(x)).to(torch.int8)
        scales[slot // page, :, slot % page] = scale
        out[name] = (rows.view(-1, kv, hd)[slot].float() * scales[slot // page, :, slot % page][..., None]).reshape(s["rows"], -1)
    return out


def _rows_of(s, name, pages):
    """Rows of K or V on these pages as fp32: [.., page, kv heads, hd]."""
    c = s["case"]
    if c["fmt"] != "q8":
        return s[name][pages].float().reshape(*pages.shape, c["page"], c["kvheads"], c["hd"])
    rows, scales = _parts(c, s[name], s["pages"])
    return rows[pages].float().mul_(scales[pages].transpose(-1, -2)[..., None])


def _load(s):
    c = s["case"]
    if own:
        _load_own(s, _stream())
        return {"k": s["kOut"], "v": s["vOut"]}
    page, start = c["page"], s["rowStart"].long()
    row = torch.arange(s["rows"], device=start.device)
    place = (s["lens"].long() - start[1:])[s["request"]] + row
    where = s["table"][s["request"], place // page].long()
    out = {}
    for name, pool in (("k", "K"), ("v", "V")):
        if c["fmt"] != "q8":
            out[name] = s[pool][where, place % page].float()
        else:
            rows, scales = _parts(c, s[pool], s["pages"])
            out[name] = (rows[where, place % page].float() * scales[where, :, place % page][..., None]).reshape(s["rows"], -1)
    return out


def _attend(s):
    c = s["case"]
    if own:
        sl = s["slopes"]
        _done(s["paged"].Attention(s["q"].data_ptr(), s["q"].stride(0), s["K"].data_ptr(), s["V"].data_ptr(), s["table"].data_ptr(), s["out"].data_ptr(),
                                   s["out"].stride(0), 0.0, c["cap"], sl.data_ptr() if sl is not None else None, _stream()))
        return s["out"]
    h, kv, hd, page = c["heads"], c["kvheads"], c["hd"], c["page"]
    group, reqs, most = h // kv, c["reqs"], s["newMost"]
    pages = s["table"][:, :-(-s["lenMost"] // page)].long()
    length = pages.shape[1] * page
    lens, start = s["lens"].long(), s["rowStart"].long()
    fresh = start[1:] - start[:-1]
    n = torch.arange(most, device=pages.device)
    row = (start[:-1, None] + n).clamp(max=s["rows"] - 1)
    q = s["q"][row].reshape(reqs, most, kv, group, hd).permute(0, 2, 3, 1, 4).reshape(reqs, kv, group * most, hd)
    k = _rows_of(s, "K", pages).reshape(reqs, length, kv, hd).permute(0, 2, 3, 1).contiguous()
    x = torch.matmul(q, k).mul_(1.0 / math.sqrt(hd)).reshape(reqs, kv, group, most, length)
    del k
    if c["cap"]:
        x = torch.tanh(x / c["cap"]) * c["cap"]
    i = ((lens - fresh)[:, None] + n)[:, :, None]
    j = torch.arange(length, device=pages.device)[None, None, :]
    if s["slopes"] is not None:
        x = x - s["slopes"].reshape(1, kv, group, 1, 1) * (i - j).abs().float()[:, None, None]
    x = x.masked_fill(((j > i) | (j >= lens[:, None, None]))[:, None, None], -math.inf)
    x = torch.exp(x - x.amax(-1, keepdim=True))
    total = x.sum(-1, keepdim=True)
    v = _rows_of(s, "V", pages).reshape(reqs, length, kv, hd).permute(0, 2, 1, 3).contiguous()
    o = (torch.matmul(x.reshape(reqs, kv, group * most, length), v) / total.reshape(reqs, kv, -1, 1)).reshape(reqs, kv, group, most, hd)
    at = torch.arange(s["rows"], device=pages.device) - start[s["request"]]
    return o[s["request"], :, :, at].reshape(s["rows"], h * hd)


# ---------------------------------------------------------------------------------------------------------------------
# the definition, in 64 bits
# ---------------------------------------------------------------------------------------------------------------------
def _values(s, name):
    """A whole pool as the values it stands for, a row a slot."""
    c = s["case"]
    if c["fmt"] != "q8":
        return s[name].double().reshape(-1, c["kvheads"], c["hd"])
    n = s["pages"] * c["page"] * c["kvheads"] * c["hd"]
    scale = s[name][n:].view(torch.float32).double().reshape(s["pages"], c["kvheads"], c["page"]).permute(0, 2, 1).reshape(-1, c["kvheads"], 1)
    return s[name][:n].view(torch.int8).double().reshape(-1, c["kvheads"], c["hd"]) * scale


def exact(case, seed):
    s = prepare(case, seed)
    h, kv, hd, page = case["heads"], case["kvheads"], case["hd"], case["page"]
    new, cached, _, _ = _sizes(case)
    if case["op"] == "store":
        where, half = s["positions"].long(), hd // 2
        turn = torch.complex(s["cos"].double()[where], s["sin"].double()[where])[:, None]

        def turned(x):
            x = x.double().reshape(s["rows"], -1, hd)
            z = torch.complex(x[..., :half].contiguous(), x[..., half:].contiguous()) * turn
            return torch.cat((z.real, z.imag), -1)

        def held(x):
            """An fp32 row as 8 bits hold it: whole multiples of a 127th of its greatest size, that step in fp32."""
            x = x.float().double()
            step = (x.abs().max(-1, keepdim=True).values / 127.0).float().double()
            whole = torch.trunc(x / step)
            whole = whole + torch.where((x - whole * step).abs() * 2 >= step, torch.sign(x), torch.zeros_like(x))
            return (whole * step).reshape(s["rows"], -1)

        return {"q": turned(s["q"]).reshape(s["rows"], -1), "k": held(turned(s["k"])), "v": held(s["v"].reshape(s["rows"], kv, hd))}
    K, V = _values(s, "K"), _values(s, "V")
    if case["op"] == "load":
        at = torch.cat([s["table"][r].long()[torch.arange(c, n + c, device=K.device) // page] * page + torch.arange(c, n + c, device=K.device) % page
                        for r, (n, c) in enumerate(zip(new, cached))])
        return {"k": K[at].reshape(s["rows"], -1), "v": V[at].reshape(s["rows"], -1)}
    out, row = torch.empty(s["q"].shape, dtype=torch.float64, device=K.device), 0
    for r, (n, c) in enumerate(zip(new, cached)):
        at = torch.arange(n + c, device=K.device)
        place = s["table"][r].long()[at // page] * page + at % page
        here = torch.arange(c, n + c, device=K.device)[:, None]
        for x in range(h):
            y = s["q"][row:row + n, x * hd:x * hd + hd].double() @ K[place, x // (h // kv)].T / hd ** 0.5
            if case["cap"]:
                y = case["cap"] * torch.tanh(y / case["cap"])
            if case["slopes"]:
                y = y - float(s["slopes"][x]) * (here - at).abs()
            y[(at > here).expand_as(y)] = -math.inf
            out[row:row + n, x * hd:x * hd + hd] = torch.softmax(y, -1) @ V[place, x // (h // kv)]
        row += n
    return out
