"""The timed work of serving several requests out of one paged KV cache (mongoose_amd.engine, HIPPaged):

  tables     block tables, slot maps and row offsets of a step from the requests' lengths, with the plan of the attention that
             follows                                                                    HIPPaged.Tables, HIPPaged.Plan
  store      rotary positions on q and k, K and V rows into the pages of the slot map   HIPPaged.Store
  attention  new tokens of every request (one or many) over the request's pages, with a tanh cap, a bias by distance, a window
             or a prefix where asked for                                                HIPPaged.Attention

`own` false: the same in elementary torch operations, 32 bits, the requests of a batch padded to the longest.  Rows are fp32 and
caches fp32 or fp16, as everywhere in this framework; lengths come from the case, values from the seed.
"""
import math
import random

import torch

own = False

_SHAPES = ((32, 8, 128), (32, 4, 64), (14, 2, 64), (8, 8, 64))       # heads, KV heads, head size of the benchmark configurations
_MOST = 2048 * 32 * 16384                                            # scores of the largest attention, padded
_TABLES = dict(op="tables", heads=32, kvheads=8, hd=128, f16=True)


# ---------------------------------------------------------------------------------------------------------------------
# cases
# ---------------------------------------------------------------------------------------------------------------------
def _attention(heads, kvheads, hd, f16, page, reqs, new, cached, singles=0.0, cap=0.0, window=0, slopes=False, prefix=0):
    return {"op": "attention", "heads": heads, "kvheads": kvheads, "hd": hd, "f16": f16, "page": page, "reqs": reqs,
            "new_lo": new[0], "new_hi": new[1], "cached_lo": cached[0], "cached_hi": cached[1], "singles": singles, "cap": cap,
            "window": window, "slopes": slopes, "prefix": prefix}


def listed():
    return [
        # a decode step of a busy server: a token for each of 64 requests, some of them just finished
        dict(_TABLES, name="tables-tokens", page=16, reqs=64, new_lo=1, new_hi=1, len_hi=4000, ended=0.05, width=256),
        # prompts that arrive together with running requests
        dict(_TABLES, name="tables-prompts", page=32, reqs=301, new_lo=1, new_hi=120, len_hi=7000, ended=0.1, width=256),
        # the rows of a decode step of the 0.5B shape
        {"name": "store-tokens", "op": "store", "heads": 14, "kvheads": 2, "hd": 64, "f16": False, "page": 16, "rows": 48},
        # a prompt's chunk of the 8B shape
        {"name": "store-chunk", "op": "store", "heads": 32, "kvheads": 8, "hd": 128, "f16": True, "page": 64, "rows": 4096},
        # one user, a short conversation: all latency
        dict(_attention(14, 2, 64, False, 16, 1, (1, 1), (500, 500)), name="token-short"),
        # a batch of conversations of very different lengths, 8B shape
        dict(_attention(32, 8, 128, True, 16, 48, (1, 1), (100, 8000)), name="token-batch"),
        # one user with a book in the cache
        dict(_attention(32, 8, 128, True, 64, 1, (1, 1), (120001, 120001)), name="token-long"),
        # a chunk of a long prompt: the matrix cores' case
        dict(_attention(32, 8, 128, True, 64, 1, (2048, 2048), (14336, 14336)), name="chunk-long"),
        # fresh prompts of odd lengths, 1.1B shape, the default cache format
        dict(_attention(32, 4, 64, False, 16, 5, (90, 700), (0, 0)), name="prompts-f32"),
        # running requests beside the chunks of two or three prompts
        dict(_attention(32, 8, 128, True, 32, 12, (100, 257), (30, 4000), singles=0.7), name="mixed"),
        # capped scores over a sliding window
        dict(_attention(32, 8, 128, True, 32, 4, (300, 600), (2000, 3500), cap=50.0, window=1024), name="capped-window"),
        # a bias by distance, shared prefixes seen both ways, a few drafted tokens a request; toy shape
        dict(_attention(8, 8, 64, False, 16, 6, (3, 3), (200, 1900), slopes=True, prefix=64), name="distance-prefix"),
    ]


def _between(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(("tables", "store", "attention", "attention", "attention", "attention"))
    page = rng.choice((8, 16, 32, 64, 128))
    if op == "tables":
        hi = rng.choice((1, 1, _between(rng, 2, 150)))
        return dict(_TABLES, page=page, reqs=_between(rng, 1, 400), new_lo=1, new_hi=hi, len_hi=_between(rng, 40, 7000),
                    ended=rng.choice((0.0, 0.1, 0.4)), width=-(-8000 // page))
    heads, kvheads, hd = rng.choice(_SHAPES)
    if op == "store":
        return {"op": "store", "heads": heads, "kvheads": kvheads, "hd": hd, "f16": rng.random() < 0.5, "page": page,
                "rows": _between(rng, 1, 4096)}
    while True:
        reqs, new = _between(rng, 1, 48), rng.choice((1, 1, _between(rng, 2, 2048)))
        cached = _between(rng, 1, 60000)
        if reqs * heads * new * (cached + new) <= _MOST and reqs * (cached + new) <= 400000:
            break
    mask = rng.choice(("", "", "", "cap", "window", "slopes", "prefix"))
    return _attention(heads, kvheads, hd, rng.random() < 0.6, page, reqs, (rng.choice((1, new)), new), (rng.choice((0, cached // 2, cached)), cached),
                      singles=rng.choice((0.0, 0.5)), cap=rng.choice((20.0, 50.0)) if mask == "cap" else 0.0,
                      window=_between(rng, 16, 4096) if mask == "window" else 0, slopes=mask == "slopes",
                      prefix=_between(rng, 2, 300) if mask == "prefix" else 0)


def _sizes(case):
    """What the case fixes of its batch: (new tokens, cached tokens, prefix) of every request; the same for every seed."""
    rng = random.Random(repr(sorted((k, v) for k, v in case.items() if k != "name")))
    new, cached = [], []
    for _ in range(case["reqs"]):
        n = rng.randint(case["new_lo"], case["new_hi"])
        if case["op"] == "tables":
            c = rng.randint(0, case["len_hi"])
            n = -1 if rng.random() < case["ended"] else n
        else:
            c = rng.randint(case["cached_lo"], case["cached_hi"])
            n = 1 if rng.random() < case["singles"] else n
        new.append(n)
        cached.append(c)
    prefix = [min(rng.randint(1, 2 * case["prefix"]), n + c) for n, c in zip(new, cached)] if case.get("prefix") else [0] * case["reqs"]
    return new, cached, prefix


def _seen(n, c, window, prefix):
    """Pairs of a new token and a position that it sees."""
    total = 0
    for i in range(c, c + n):
        first = max(0, i - window + 1) if window else 0
        total += i + 1 - first + max(0, min(prefix, first)) + max(0, prefix - i - 1)
    return total


def work(case):
    h, kv, hd, cache = case["heads"], case["kvheads"], case["hd"], 2 if case["f16"] else 4
    if case["op"] == "store":
        return {"bytes": case["rows"] * (2 * h * hd * 4 + 2 * kv * hd * (4 + cache) + hd * 4 + 8), "flops": case["rows"] * (h + kv) * hd * 3}
    new, cached, prefix = _sizes(case)
    if case["op"] == "tables":
        p = case["page"]
        rows = sum(n for n in new if n > 0)
        pages = sum(-(-(n + c) // p) - -(-c // p) if n >= 0 else -(-c // p) for n, c in zip(new, cached))
        return {"bytes": 4 * (4 * case["reqs"] + 2 * rows + 2 * pages), "flops": 0}
    rows = sum(new)
    read = sum(n + c - (max(0, c - case["window"] + 1) if case["window"] else 0) for n, c in zip(new, cached))
    pairs = sum(_seen(n, c, case["window"], p) for n, c, p in zip(new, cached, prefix))
    return {"bytes": 2 * rows * h * hd * 4 + 2 * read * kv * hd * cache, "flops": 4 * hd * h * pairs}


# ---------------------------------------------------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------------------------------------------------
def _ints(values, dev):
    return torch.tensor(values, dtype=torch.int32, device=dev)


def _handle(s, rows, width):
    """The handle that a server keeps for a model's attention; `width`: pages of a request's row of the block table."""
    from mongoose_amd import engine as E
    c = s["case"]
    s["paged"] = E.NewHIPPaged(E.NewHIP(), c["heads"], c["kvheads"], c["hd"], c["page"], s["pages"], 1 if c["f16"] else 0, c.get("reqs", 1), rows, width * c["page"])
    if s["paged"] is None:
        raise RuntimeError(E.last_error())


def _done(rc):
    if rc:
        from mongoose_amd import engine as E
        raise RuntimeError(E.last_error())


def _stream():
    return torch.cuda.current_stream().cuda_stream


def prepare(case, seed):
    dev = torch.device("cuda")
    g = torch.Generator(device=dev)
    g.manual_seed(seed)
    s = {"case": case, "seed": seed}
    page, hd = case["page"], case["hd"]
    if case["op"] == "store":
        return _prepare_store(s, g, dev)
    new, cached, prefix = _sizes(case)
    if case["op"] == "tables":
        return _prepare_tables(s, g, dev, new, cached)
    lens = [n + c for n, c in zip(new, cached)]
    rows, most = sum(new), max(lens)
    width = -(-most // page) + 1
    used = sum(-(-x // page) for x in lens)
    s["pages"] = used + used // 8 + 1                                    # a pool that is nearly full, in the order of its use
    order = torch.randperm(s["pages"], generator=g, device=dev)[:used].to(torch.int32)
    at = torch.arange(width, device=dev)
    count = torch.tensor([-(-x // page) for x in lens], device=dev)
    first = torch.cumsum(count, 0) - count
    s["table"] = torch.where(at < count[:, None], order[(first[:, None] + at).clamp(max=used - 1)], 0).to(torch.int32).contiguous()
    s["rowStart"] = _ints([sum(new[:i]) for i in range(len(new) + 1)], dev)
    s["lens"] = _ints(lens, dev)
    s["prefix"] = _ints(prefix, dev) if case["prefix"] else None
    s["rows"], s["newMost"], s["lenMost"] = rows, max(new), most
    s["request"] = torch.repeat_interleave(torch.arange(len(new), device=dev), torch.tensor(new, device=dev))
    kind = torch.float16 if case["f16"] else torch.float32
    size = (s["pages"], page, case["kvheads"] * hd)
    channel = torch.exp(0.4 * torch.randn(size[2], generator=g, device=dev))          # channels of K differ in size, as trained ones do
    s["K"] = torch.randn(size, generator=g, device=dev, dtype=kind).mul_(channel.to(kind))
    s["V"] = torch.randn(size, generator=g, device=dev, dtype=kind)
    s["q"] = 1.5 * torch.randn((rows, case["heads"] * hd), generator=g, device=dev)
    s["slopes"] = torch.exp2(-8.0 * torch.arange(1, case["heads"] + 1, device=dev) / case["heads"]) if case["slopes"] else None
    if own:
        s["out"] = torch.empty_like(s["q"])
        _handle(s, rows, width)
        p = s["prefix"]
        _done(s["paged"].Plan(s["rowStart"].data_ptr(), s["lens"].data_ptr(), case["reqs"], rows, case["window"], p.data_ptr() if p is not None else None, _stream()))
    return s


def _prepare_tables(s, g, dev, new, cached):
    c = s["case"]
    page, width = c["page"], c["width"]
    held = [-(-x // page) for x in cached]
    need = sum(-(-(n + x) // page) - h for n, x, h in zip(new, cached, held) if n >= 0)
    used = sum(held)
    s["pages"] = used + need + max(8, used // 16)
    order = torch.randperm(s["pages"], generator=g, device=dev).to(torch.int32)
    at = torch.arange(width, device=dev)
    count = torch.tensor(held, device=dev)
    first = torch.cumsum(count, 0) - count
    s["table"] = torch.where(at < count[:, None], order[(first[:, None] + at).clamp(max=s["pages"] - 1)], 0).to(torch.int32).contiguous()
    head = s["seed"] % s["pages"]
    s["ring"] = torch.roll(torch.cat((order[used:], torch.zeros(used, dtype=torch.int32, device=dev))), head)
    s["ringState"] = _ints([head, s["pages"] - used], dev)
    s["new"], s["lens"] = _ints(new, dev), _ints(cached, dev)
    s["rows"] = (sum(n for n in new if n > 0) + 63) // 64 * 64                        # rows as a captured step has them: some are left over
    for name, n in (("lensOut", c["reqs"]), ("ringStateOut", 2), ("rowStart", c["reqs"] + 1), ("slots", s["rows"]), ("positions", s["rows"]), ("counts", 4)):
        s[name] = torch.zeros(n, dtype=torch.int32, device=dev)
    if own:
        _handle(s, max(1, s["rows"]), width)
    return s


def _prepare_store(s, g, dev):
    c = s["case"]
    h, kv, hd, rows, page = c["heads"], c["kvheads"], c["hd"], c["rows"], c["page"]
    s["pages"] = -(-rows * 5 // (4 * page)) + 1
    qkv = torch.randn((rows, (h + 2 * kv) * hd), generator=g, device=dev)             # rows of one projection
    s["q"], s["k"], s["v"] = qkv[:, :h * hd], qkv[:, h * hd:(h + kv) * hd], qkv[:, (h + kv) * hd:]
    kind = torch.float16 if c["f16"] else torch.float32
    s["K"] = torch.randn((s["pages"], page, kv * hd), generator=g, device=dev, dtype=kind)
    s["V"] = torch.randn((s["pages"], page, kv * hd), generator=g, device=dev, dtype=kind)
    s["slots"] = torch.randperm(s["pages"] * page, generator=g, device=dev)[:rows].to(torch.int32)
    far = 8192
    s["positions"] = torch.randint(0, far, (rows,), generator=g, device=dev, dtype=torch.int32)
    angle = torch.arange(far, device=dev, dtype=torch.float64)[:, None] * 5e5 ** (-torch.arange(hd // 2, device=dev, dtype=torch.float64) * 2 / hd)
    s["cos"], s["sin"], s["far"] = torch.cos(angle).float(), torch.sin(angle).float(), far
    s["qOut"] = torch.empty((rows, h * hd), device=dev)
    if own:
        _handle(s, rows, s["pages"])
    return s


# ---------------------------------------------------------------------------------------------------------------------
# one pass
# ---------------------------------------------------------------------------------------------------------------------
def run(s):
    return {"tables": _tables, "store": _store, "attention": _attend}[s["case"]["op"]](s)


def _tables(s):
    c = s["case"]
    if own:
        p, st = s["paged"], _stream()
        at = {k: s[k].data_ptr() for k in ("new", "lens", "lensOut", "table", "ring", "ringState", "ringStateOut", "rowStart", "slots", "positions", "counts")}
        _done(p.Tables(at["new"], c["reqs"], at["lens"], at["lensOut"], at["table"], at["ring"], at["ringState"], at["ringStateOut"], s["rows"],
                       at["rowStart"], at["slots"], at["positions"], at["counts"], st))
        _done(p.Plan(at["rowStart"], at["lensOut"], c["reqs"], s["rows"], 0, None, st))
        return {k: s[k] for k in ("table", "ring", "lensOut", "ringStateOut", "rowStart", "slots", "positions", "counts")}
    page, n, dev = c["page"], s["pages"], s["new"].device
    lens, new = s["lens"].long(), s["new"].long()
    ended, fresh = new < 0, new.clamp(min=0)
    held = (lens + page - 1) // page
    taken = (lens + fresh + page - 1) // page - held
    start = torch.cat((torch.zeros(1, dtype=torch.long, device=dev), torch.cumsum(fresh, 0)))
    before = torch.cumsum(taken, 0) - taken
    head, free = s["ringState"][0].long(), s["ringState"][1].long()
    i = torch.arange(s["rows"], device=dev)
    r = torch.searchsorted(start[1:], i, right=True).clamp(max=c["reqs"] - 1)
    live = i < start[-1]
    pos = lens[r] + i - start[r]
    # the pages taken: entry e of request r with held <= e < held + taken
    e = torch.arange(c["width"], device=dev)
    isNew = (e >= held[:, None]) & (e < (held + taken)[:, None])
    table = torch.where(isNew, s["ring"][(head + before[:, None] + e - held[:, None]).clamp(min=0) % n], s["table"])
    slot = table[r, (pos // page).clamp(max=c["width"] - 1)].long() * page + pos % page
    # the pages given back, behind the free ones
    back = ended[:, None] & (e < held[:, None])
    order = torch.cumsum(back.reshape(-1), 0) - 1
    given = back.sum()
    ring = torch.cat((s["ring"], torch.zeros(1, dtype=torch.int32, device=dev)))
    ring[torch.where(back.reshape(-1), (head + free + order) % n, n)] = table.reshape(-1)
    s["table"].copy_(table)
    s["ring"].copy_(ring[:n])
    out = {"table": s["table"], "ring": s["ring"], "lensOut": torch.where(ended, 0, lens + fresh),
           "ringStateOut": torch.stack(((head + taken.sum()) % n, free - taken.sum() + given)), "rowStart": start,
           "slots": torch.where(live, slot, -1), "positions": torch.where(live, pos, -1),
           "counts": torch.stack((start[-1], taken.sum(), given, torch.zeros_like(given)))}
    return {k: v.to(torch.int32) for k, v in out.items()}


def _store(s):
    c = s["case"]
    if own:
        _done(s["paged"].Store(s["q"].data_ptr(), s["k"].data_ptr(), s["v"].data_ptr(), s["q"].stride(0), s["k"].stride(0), s["v"].stride(0), s["qOut"].data_ptr(),
                               s["qOut"].stride(0), s["K"].data_ptr(), s["V"].data_ptr(), s["slots"].data_ptr(), s["positions"].data_ptr(), c["rows"],
                               s["cos"].data_ptr(), s["sin"].data_ptr(), s["far"], _stream()))
        return {k: s[k] for k in ("qOut", "K", "V")}
    hd, at = c["hd"], s["positions"].long()
    cos, sin = s["cos"][at][:, None, :], s["sin"][at][:, None, :]

    def turned(x):
        a, b = x.reshape(c["rows"], -1, 2, hd // 2).unbind(2)
        return torch.stack((a * cos - b * sin, a * sin + b * cos), 2).reshape(c["rows"], -1)

    slot = s["slots"].long()
    s["K"].view(-1, c["kvheads"] * hd)[slot] = turned(s["k"]).to(s["K"].dtype)
    s["V"].view(-1, c["kvheads"] * hd)[slot] = s["v"].to(s["V"].dtype)
    s["qOut"].copy_(turned(s["q"]))
    return {k: s[k] for k in ("qOut", "K", "V")}


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
    k = s["K"][pages].float().reshape(reqs, length, kv, hd).permute(0, 2, 3, 1).contiguous()
    x = torch.matmul(q, k).mul_(1.0 / math.sqrt(hd)).reshape(reqs, kv, group, most, length)
    del k
    if c["cap"]:
        x = torch.tanh(x / c["cap"]) * c["cap"]
    i = ((lens - fresh)[:, None] + n)[:, :, None]
    j = torch.arange(length, device=pages.device)[None, None, :]
    if s["slopes"] is not None:
        x = x - s["slopes"].reshape(1, kv, group, 1, 1) * (i - j).abs().float()[:, None, None]
    seen = j <= i
    if c["window"]:
        seen = seen & (j > i - c["window"])
    if s["prefix"] is not None:
        seen = seen | (j < s["prefix"].long()[:, None, None])
    seen = (seen & (j < lens[:, None, None]))[:, None, None]
    x = x.masked_fill(~seen, -math.inf)
    x = torch.exp(x - x.amax(-1, keepdim=True))
    total = x.sum(-1, keepdim=True)
    v = s["V"][pages].float().reshape(reqs, length, kv, hd).permute(0, 2, 1, 3).contiguous()
    o = (torch.matmul(x.reshape(reqs, kv, group * most, length), v) / total.reshape(reqs, kv, -1, 1)).reshape(reqs, kv, group, most, hd)
    at = torch.arange(s["rows"], device=pages.device) - start[s["request"]]
    return o[s["request"], :, :, at].reshape(s["rows"], h * hd)


# ---------------------------------------------------------------------------------------------------------------------
# the definition, in 64 bits
# ---------------------------------------------------------------------------------------------------------------------
def exact(case, seed):
    s = prepare(case, seed)
    hd, page = case["hd"], case["page"]
    if case["op"] == "tables":
        return _exact_tables(s)
    if case["op"] == "store":
        K, V = s["K"].double().reshape(-1, case["kvheads"], hd), s["V"].double().reshape(-1, case["kvheads"], hd)
        where, slot, half = s["positions"].long(), s["slots"].long(), hd // 2
        turn = torch.complex(s["cos"].double()[where], s["sin"].double()[where])[:, None]
        rotated = []
        for x in (s["q"], s["k"]):
            x = x.double().reshape(case["rows"], -1, hd)
            z = torch.complex(x[..., :half].contiguous(), x[..., half:].contiguous()) * turn
            rotated.append(torch.cat((z.real, z.imag), -1))
        K[slot], V[slot] = rotated[1], s["v"].double().reshape(case["rows"], -1, hd)
        return {"qOut": rotated[0].reshape(case["rows"], -1), "K": K.reshape(s["K"].shape), "V": V.reshape(s["V"].shape)}
    new, cached, prefix = _sizes(case)
    group = case["heads"] // case["kvheads"]
    out, row = torch.empty(s["q"].shape, dtype=torch.float64, device=s["q"].device), 0
    for r, (n, c) in enumerate(zip(new, cached)):
        at = torch.arange(n + c, device=out.device)
        place = s["table"][r].long()[at // page] * page + at % page
        here = torch.arange(c, n + c, device=out.device)[:, None]
        hidden = at > here
        if case["window"]:
            hidden |= at <= here - case["window"]
        hidden &= at >= prefix[r]
        for h in range(case["heads"]):
            cols = slice(h // group * hd, h // group * hd + hd)
            y = s["q"][row:row + n, h * hd:h * hd + hd].double() @ s["K"].reshape(-1, case["kvheads"] * hd)[place, cols].double().T / hd ** 0.5
            if case["cap"]:
                y = case["cap"] * torch.tanh(y / case["cap"])
            if case["slopes"]:
                y = y - float(s["slopes"][h]) * (here - at).abs()
            y[hidden] = -math.inf
            out[row:row + n, h * hd:h * hd + hd] = torch.softmax(y, -1) @ s["V"].reshape(-1, case["kvheads"] * hd)[place, cols].double()
        row += n
    return out


def _exact_tables(s):
    c = s["case"]
    page, n = c["page"], s["pages"]
    new, lens, table, ring = (s[k].tolist() for k in ("new", "lens", "table", "ring"))
    head, free = s["ringState"].tolist()
    queue = [ring[(head + j) % n] for j in range(free)]
    start, slots, positions, taken, given = [0], [], [], 0, []
    for r, x in enumerate(new):
        for pos in range(lens[r], lens[r] + max(0, x)):
            if pos % page == 0:
                table[r][pos // page] = queue[taken]
                taken += 1
            slots.append(table[r][pos // page] * page + pos % page)
            positions.append(pos)
        if x < 0:
            given += table[r][:-(-lens[r] // page)]
        lens[r] = lens[r] + x if x >= 0 else 0
        start.append(len(slots))
    for j, p in enumerate(given):
        ring[(head + free + j) % n] = p
    rest = s["rows"] - len(slots)
    out = {"table": table, "ring": ring, "lensOut": lens, "ringStateOut": [(head + taken) % n, free - taken + len(given)], "rowStart": start,
           "slots": slots + [-1] * rest, "positions": positions + [-1] * rest, "counts": [start[-1], taken, len(given), 0]}
    return {k: torch.tensor(v, dtype=torch.int32) for k, v in out.items()}
