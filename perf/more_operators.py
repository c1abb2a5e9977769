"""What the performance of serving many sequences from a small cache is measured on: rows kept in four bits and the attention over them, pages handed out
on the GPU, and rotary positions; each in a plain form (elementary torch operations in 32 bits) and through the framework's entry points.

Kinds of case
  rows     KvCache.write, KvCache.read with kind "uint4": rows of keys and values into a paged cache as codes of four bits, with a scale and a least value in bf16
           for each token and head (x ~ least + scale * code), and the same rows read back
  attend   KvCache.attend over such a cache: attention of one new row per sequence, where asked with the new row's key and value appended first (and then read back)
  pages    KvPages.grow, KvPages.shrink: requests' new rows get pages from a free list, slots and positions, from counts that are on the GPU, and are given back
  rope     Rotary: rows of queries and keys turned by their positions, in either layout, all or a part of a head, frequencies as they are or scaled for long contexts
"""
import math

import torch

own = False  # False: the plain forms; True: the framework's operators

D = 128  # width of a head
THETA = 5000000.0
FLOOR = 2.0 ** -100  # the least spread that a scale is made of
DTYPES = {"bf16": torch.bfloat16, "fp32": torch.float32}


def listed():
    return [
        # the key and value rows of one short prompt: the smallest write, bound by latency
        {"name": "rows_prompt_77", "kind": "rows", "rows": 77, "kv_heads": 8, "page": 16, "used": 0.5},
        # the rows of the largest sequence the framework is measured on
        {"name": "rows_long_16640", "kind": "rows", "rows": 16640, "kv_heads": 8, "page": 64, "used": 0.9},
        # one short prompt continued by a row: latency only
        {"name": "attend_one_85", "kind": "attend", "batch": 1, "heads": 32, "kv_heads": 8, "least": 85, "most": 85, "page": 16, "append": True, "lse": False},
        # a served batch of ragged lengths in small pages, some sequences empty, a key head for every two query heads
        {"name": "attend_batch_37", "kind": "attend", "batch": 37, "heads": 16, "kv_heads": 8, "least": 0, "most": 1999, "page": 32, "append": False, "lse": True},
        # one very long sequence: few (sequence, head) pairs, so the length has to be split over the whole GPU
        {"name": "attend_long_100003", "kind": "attend", "batch": 1, "heads": 32, "kv_heads": 8, "least": 100003, "most": 100003, "page": 64, "append": False,
         "lse": True},
        # a full server of many long sequences, the new rows appended: bound by memory alone, if the arithmetic keeps up
        {"name": "attend_server_96", "kind": "attend", "batch": 96, "heads": 32, "kv_heads": 8, "least": 300, "most": 5400, "page": 64, "append": True, "lse": False},
        # one step of a served batch: a row for each of some of the open sequences
        {"name": "pages_step_24", "kind": "pages", "batch": 24, "open": 32, "old": 2100, "new": 1, "page": 16, "least": 1},
        # requests that come in together: prompts of ragged lengths, some of them continuing older rows
        {"name": "pages_prompts_61", "kind": "pages", "batch": 61, "open": 61, "old": 300, "new": 1500, "page": 64, "least": 0},
        # a large server's prompts, small pages: many rows and many sequences
        {"name": "pages_server_1000", "kind": "pages", "batch": 1000, "open": 1024, "old": 700, "new": 300, "page": 16, "least": 0},
        # the queries and keys of a step of a served batch
        {"name": "rope_step_24", "kind": "rope", "rows": 24, "heads": 32, "kv_heads": 8, "head": 128, "rot": 128, "layout": "half", "scaling": "none", "far": 5400,
         "type": "bf16"},
        # an odd number of rows at far positions, half of a head turned in pairs of neighbours, frequencies scaled by parts
        {"name": "rope_part_4111", "kind": "rope", "rows": 4111, "heads": 16, "kv_heads": 4, "head": 128, "rot": 64, "layout": "interleaved", "scaling": "yarn",
         "far": 1000003, "type": "fp32"},
        # the largest sequence
        {"name": "rope_long_16640", "kind": "rope", "rows": 16640, "heads": 32, "kv_heads": 8, "head": 128, "rot": 128, "layout": "half", "scaling": "linear",
         "far": 16640, "type": "bf16"},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["rows", "attend", "attend", "attend", "pages", "rope"])
    if kind == "rows":
        heads = rng.choice([1, 2, 4, 8, 8, 16])
        return {"kind": kind, "rows": _log(rng, 1, 16640 * 8 // max(8, heads)), "kv_heads": heads, "page": rng.choice([16, 32, 48, 64, 128]),
                "used": round(rng.uniform(0.3, 0.95), 2)}
    if kind == "attend":
        kv_heads = rng.choice([1, 2, 4, 8, 8, 16])
        heads = kv_heads * rng.choice([1, 2, 3, 4, 4, 7, 8, 16][: 8 if kv_heads <= 4 else 7])
        batch = _log(rng, 1, 128)
        most = _log(rng, 1, min(100003, 2000000 // (batch * kv_heads)))
        append = rng.random() < 0.5
        least = rng.choice([most, max(1, most // 2), 1, 0])
        return {"kind": kind, "batch": batch, "heads": heads, "kv_heads": kv_heads, "least": max(1, least) if append else least, "most": most,
                "page": rng.choice([16, 32, 48, 64, 128]), "append": append, "lse": rng.random() < 0.5}
    if kind == "pages":
        batch = _log(rng, 1, 1000)
        new = rng.choice([1, 1, _log(rng, 2, min(4000, 300000 // batch))])
        return {"kind": kind, "batch": batch, "open": batch + rng.choice([0, 0, _log(rng, 1, 40)]), "old": _log(rng, 1, min(5400, 2000000 // batch)), "new": new,
                "page": rng.choice([16, 32, 48, 64, 128]), "least": 1 if new == 1 else rng.choice([0, 1])}
    head = rng.choice([64, 72, 96, 128, 128, 128, 256])
    heads, kv_heads = rng.choice([(32, 8), (16, 16), (8, 1), (4, 2), (7, 1), (12, 4)])
    type_ = rng.choice(["bf16", "bf16", "fp32"])
    size = (heads + kv_heads) * head * (1 if type_ == "bf16" else 2)
    return {"kind": kind, "rows": _log(rng, 1, 16640 * 40 * 128 // max(size, 40 * 128)), "heads": heads, "kv_heads": kv_heads, "head": head,
            "rot": rng.choice([head, head, head // 2, 2 * rng.randint(1, head // 2)]), "layout": rng.choice(["half", "interleaved"]),
            "scaling": rng.choice(["none", "linear", "ntk", "yarn"]), "far": _log(rng, 100, 1000003), "type": type_}


# ------------------------------------------------------------------ sizes
def _spread(count, a, b):
    """So many sizes between a and b, both included."""
    return [a + int((0.5 + 0.6180339887498949 * i) % 1.0 * (b - a + 1)) for i in range(count)]


def _lens(case):
    """Rows of each sequence, the new one included."""
    return _spread(case["batch"], case["least"], case["most"])


def _requests(case):
    """(rows that each open sequence has, new rows of each one of the batch, which of the open ones those are)."""
    old = [(n * 7919) % (case["old"] + 1) for n in range(1, case["open"] + 1)]
    return old, _spread(case["batch"], case["least"], case["new"]), [(5 * i + 3) % case["open"] if case["open"] % 5 else i for i in range(case["batch"])]


def _width(case):
    return -(-(case["old"] + case["new"]) // case["page"])


ROW = 2 * (D // 2 + 4)  # bytes of a token's key and value of a head: codes of four bits, a scale and a least value


def work(case):
    if case["kind"] == "rows":
        # rows in, codes and scales out, codes and scales in, rows out; the slots twice
        io = case["rows"] * 2 * case["kv_heads"] * D * 2
        return {"bytes": 2 * io + 2 * case["rows"] * case["kv_heads"] * ROW + 16 * case["rows"], "flops": 0}
    if case["kind"] == "attend":
        total, new = sum(_lens(case)), case["batch"] * case["kv_heads"] * (ROW + 4 * D + ROW + 4 * D) if case["append"] else 0
        io = case["batch"] * case["heads"] * (2 * D * 2 + (4 if case["lse"] else 0))
        tables = 4 * sum(-(-n // case["page"]) + 1 for n in _lens(case))
        return {"bytes": total * case["kv_heads"] * ROW + new + io + tables, "flops": 4 * D * case["heads"] * total}
    if case["kind"] == "pages":
        # counts, names, lengths in and out, rows' slots and positions, tables of the batch; pages taken and given back
        old, new, names = _requests(case)
        taken = sum(-(-(old[s] + n) // case["page"]) - -(-old[s] // case["page"]) for s, n in zip(names, new))
        tables = sum(-(-(old[s] + n) // case["page"]) for s, n in zip(names, new))
        return {"bytes": 12 * sum(new) + 4 * case["batch"] * (8 + _width(case)) + 4 * (tables + 6 * taken), "flops": 0}
    n = case["rows"] * (case["heads"] + case["kv_heads"]) * case["head"]
    return {"bytes": 2 * n * DTYPES[case["type"]].itemsize + 8 * case["rows"], "flops": 3 * n * case["rot"] // case["head"]}


# ------------------------------------------------------------------ inputs
def _gen(seed, salt=0):
    g = torch.Generator(device="cuda")
    g.manual_seed(int(seed) * 131 + salt)
    return g


def _normal(shape, g, std=1.0, dtype=torch.bfloat16):
    return torch.empty(shape, dtype=dtype, device="cuda").normal_(0.0, std, generator=g)


def _quantised(x):
    """Codes of rows x [..., D] and the pairs (scale, least) [..., 2] that they stand for values with."""
    x = x.float()
    least, spread = x.amin(-1) + 0.0, x.amax(-1) - x.amin(-1)
    scale = torch.where(spread >= FLOOR, spread * (1.0 / 15.0), 0.0).to(torch.bfloat16)
    inv = torch.where(scale > 0, torch.ones_like(spread) / scale.float(), 0.0)
    codes = ((x - least[..., None]) * inv[..., None]).round().to(torch.uint8)
    return codes, torch.stack([scale, least.to(torch.bfloat16)], -1)


def _packed(codes):
    """Two codes to a byte, the first one in the low bits."""
    return codes[..., ::2] | codes[..., 1::2] << 4


def _values(packed, scales):
    """What packed codes and scales stand for, in 32 bits."""
    codes = torch.stack([packed & 15, packed >> 4], -1).flatten(-2).float()
    return scales[..., 1:].float() + codes * scales[..., :1].float()


def _cache(case, pages, g, filled):
    """A cache of so many pages; filled: with keys that have a few strong channels, as projected keys have, and plain values."""
    shape = (pages, case["kv_heads"], case["page"])
    s = {}
    for name in ("k", "v"):
        s[name] = torch.zeros(shape + (D // 2,), dtype=torch.uint8, device="cuda")
        s[name + "_scale"] = torch.zeros(shape + (2,), dtype=torch.bfloat16, device="cuda")
        if not filled:
            continue
        strong = torch.ones(D, dtype=torch.bfloat16, device="cuda")
        if name == "k":
            strong[::17] = 4.0
        step = max(1, (1 << 25) // (shape[1] * shape[2] * D))
        for at in range(0, pages, step):
            codes, scales = _quantised(_normal((min(step, pages - at),) + shape[1:] + (D,), g) * strong)
            s[name][at:at + step], s[name + "_scale"][at:at + step] = _packed(codes), scales
    return s


def _frequencies(case, device):
    """Radians a position of each pair, in 64 bits, and what the turned values are multiplied by."""
    rot, far = case["rot"], 8.0
    i = torch.arange(rot // 2, dtype=torch.float64, device=device)
    if case["scaling"] == "ntk":
        return (THETA * far ** (rot / max(rot - 2, 1))) ** (-2.0 * i / rot), 1.0
    freq = THETA ** (-2.0 * i / rot)
    if case["scaling"] == "linear":
        return freq / far, 1.0
    if case["scaling"] == "yarn":
        # as they are where a pair turns 32 times or more within the original length, divided where it turns once or less, a ramp between
        def at(turns):
            return rot * math.log(ORIGINAL / (turns * 2.0 * math.pi)) / (2.0 * math.log(THETA))

        low, high = max(math.floor(at(32.0)), 0), min(math.ceil(at(1.0)), rot - 1)
        ramp = ((i - low) / max(high - low, 0.001)).clamp(0.0, 1.0)
        return freq / far * ramp + freq * (1.0 - ramp), 0.1 * math.log(far) + 1.0
    return freq, 1.0


ORIGINAL = 16640  # the length that a scaled context was made from


def prepare(case, seed):
    g = _gen(seed)
    s = {"case": case}
    if own:
        from __graft_entry__ import load_package
        o1 = load_package()
        o1.use_torch_stream()
    if case["kind"] == "rope":
        rows, heads, kv_heads, head = case["rows"], case["heads"], case["kv_heads"], case["head"]
        # queries and keys are slices of the projections' rows (q | k | v)
        qkv = _normal((rows, (heads + 2 * kv_heads) * head), g, 1.0, DTYPES[case["type"]])
        s["q"], s["k"] = qkv[:, :heads * head].view(rows, heads, head), qkv[:, heads * head:(heads + kv_heads) * head].view(rows, kv_heads, head)
        start = torch.randint(0, max(1, case["far"] - rows + 1), (1,), generator=g, device="cuda")
        s["positions"] = (torch.arange(rows, device="cuda") + start).clamp_max(case["far"]).to(torch.int32)
        s["freq"], s["factor"] = _frequencies(case, "cuda")
        if own:
            s["rope"] = o1.Rotary(head, case["rot"], THETA, case["layout"], None if case["scaling"] == "none" else
                                  {"kind": case["scaling"], "factor": 8.0, "original": ORIGINAL})
        return s
    if case["kind"] == "pages":
        old, new, names = _requests(case)
        need = [-(-n // case["page"]) for n in old]
        pages = sum(-(-(n + case["new"]) // case["page"]) for n in old) + 5
        order = torch.randperm(pages, generator=g, device="cuda").to(torch.int32)
        table = torch.full((case["open"], _width(case)), -1, dtype=torch.int32)
        at = torch.arange(table.size(1))[None, :] < torch.tensor(need)[:, None]
        table[at] = order.cpu()[:sum(need)]
        s["table"], s["lens"] = table.cuda(), torch.tensor(old, dtype=torch.int32).cuda()
        s["free"] = torch.cat([order[sum(need):], torch.zeros(sum(need), dtype=torch.int32, device="cuda")])
        s["state"] = torch.tensor([pages - sum(need), 0], dtype=torch.int32).cuda()
        s["counts"], s["rows"] = torch.tensor(new, dtype=torch.int32).cuda(), sum(new)
        s["names"] = torch.tensor(names, dtype=torch.int32).cuda()
        s["before"] = s["lens"][s["names"].long()].contiguous()
        if own:
            s["pages"] = o1.KvPages.over(s["table"], s["lens"], s["free"], s["state"], case["page"])
        return s
    if case["kind"] == "rows":
        rows, heads, page = case["rows"], case["kv_heads"], case["page"]
        pages = -(-int(rows / case["used"] + 1) // page)
        s |= _cache(case, pages, g, False)
        # keys and values are slices of the projections' rows (q | k | v, four query heads to a key head)
        qkv = _normal((rows, 6 * heads * D), g)
        s["new_k"], s["new_v"] = (qkv[:, (4 + i) * heads * D:(5 + i) * heads * D].view(rows, heads, D) for i in (0, 1))
        s["slots"] = torch.randperm(pages * page, generator=g, device="cuda")[:rows].contiguous()
    else:
        batch, page, lens = case["batch"], case["page"], _lens(case)
        need = [-(-n // page) for n in lens]
        width, pages = max(max(need), 1), sum(need) + 3
        s |= _cache(case, pages, g, True)
        order = torch.randperm(pages, generator=g, device="cuda").to(torch.int32)
        table = torch.full((batch, width), -1, dtype=torch.int32)
        at = torch.arange(width)[None, :] < torch.tensor(need)[:, None]
        table[at] = order.cpu()[:sum(need)]
        s["pages"], s["lens"] = table.cuda(), torch.tensor(lens, dtype=torch.int32).cuda()
        qkv = _normal((batch, (case["heads"] + 2 * case["kv_heads"]) * D), g)
        q, k, v = qkv.split([case["heads"] * D, case["kv_heads"] * D, case["kv_heads"] * D], dim=1)
        s["q"] = q.view(batch, case["heads"], D)
        s["new_k"], s["new_v"] = (a.view(batch, case["kv_heads"], D) if case["append"] else None for a in (k, v))
        last = s["lens"].long() - 1
        s["slots"] = s["pages"].long().gather(1, (last.clamp_min(0) // page)[:, None])[:, 0] * page + last % page if case["append"] else None
    if own:
        s["cache"] = o1.KvCache.over(s["k"], s["v"], s["k_scale"], s["v_scale"])
    return s


# ------------------------------------------------------------------ plain forms
def _store(s):
    page, at = s["slots"] // s["case"]["page"], s["slots"] % s["case"]["page"]
    for name in ("k", "v"):
        codes, scales = _quantised(s["new_" + name])
        s[name][page, :, at], s[name + "_scale"][page, :, at] = _packed(codes), scales


def _load(s):
    page, at = s["slots"] // s["case"]["page"], s["slots"] % s["case"]["page"]
    return {name: _values(s[name][page, :, at], s[name + "_scale"][page, :, at]).to(torch.bfloat16) for name in ("k", "v")}


def _plain_rows(s):
    _store(s)
    return _load(s)


def _gathered(s, name, table, valid):
    """Rows [batch, kv_heads, width * page, D] in 32 bits, zeros where a sequence has none."""
    x = _values(s[name][table], s[name + "_scale"][table])
    x = x.permute(0, 2, 1, 3, 4).reshape(table.shape[0], s[name].shape[1], -1, D)
    return x.masked_fill_(~valid[:, None, :, None], 0.0)


def _plain_attend(s):
    case, lens = s["case"], s["lens"].long()
    table = s["pages"].long().clamp_min(0)
    if s["new_k"] is not None:
        _store(s)
    valid = torch.arange(table.shape[1] * case["page"], device="cuda")[None, :] < lens[:, None]
    k = _gathered(s, "k", table, valid)
    q = s["q"].float().reshape(case["batch"], case["kv_heads"], -1, D)
    z = (q @ k.transpose(2, 3)) * D ** -0.5
    z = z.masked_fill_(~valid[:, None, None, :], -math.inf)
    top = z.amax(-1, keepdim=True)
    p = torch.exp(z - torch.where(top == -math.inf, 0.0, top))
    total = p.sum(-1, keepdim=True)
    out = p @ _gathered(s, "v", table, valid)
    out = torch.where(total > 0, out / total, 0.0).reshape(case["batch"], case["heads"], D).to(torch.bfloat16)
    got = {"out": out}
    if case["lse"]:
        got["lse"] = (top + torch.log(total)).reshape(case["batch"], case["heads"])
    return got | (_load(s) if s["new_k"] is not None else {})


def _plain_pages(s):
    page, names, counts, rows = s["case"]["page"], s["names"].long(), s["counts"].long(), s["rows"]
    table, free, batch = s["table"], s["free"], s["names"].numel()
    # ---- rows are added
    lens, have = s["lens"][names].long(), s["state"][0].long()
    old, new = (lens + page - 1) // page, (lens + counts + page - 1) // page
    ends, starts = (new - old).cumsum(0), torch.zeros(batch + 1, dtype=torch.int32, device="cuda")
    starts[1:] = counts.cumsum(0)
    j = torch.arange(table.shape[1], device="cuda")[None, :]
    fresh = (j >= old[:, None]) & (j < new[:, None])
    taken = (have - 1 - (ends - (new - old))[:, None] - (j - old[:, None])).clamp(0, free.numel() - 1)
    pages = torch.where(fresh, free[taken], table[names])
    table[names] = pages
    which = torch.repeat_interleave(torch.arange(batch, device="cuda"), counts, output_size=rows)
    positions = torch.arange(rows, device="cuda") - starts[which] + lens[which]
    slots = pages[which, positions // page].long() * page + positions % page
    s["lens"][names] = (lens + counts).int()
    s["state"][0] -= ends[-1]
    got = {"slots": slots, "positions": positions.int(), "starts": starts, "lens": (lens + counts).int(), "pages": pages}
    # ---- and given back
    lens, have = s["lens"][names].long(), s["state"][0].long()
    old, new = (lens + page - 1) // page, (s["before"].long() + page - 1) // page
    ends = (old - new).cumsum(0)
    gone = (j >= new[:, None]) & (j < old[:, None])
    to = have + ends[-1] - 1 - (ends - (old - new))[:, None] - (j - new[:, None])
    s["free"] = torch.cat([free, free[:1]]).scatter_(0, torch.where(gone, to, free.numel()).flatten(), torch.where(gone, pages, 0).flatten())[:-1]
    table[names] = torch.where(gone, -1, pages)
    s["lens"][names] = s["before"]
    s["state"][0] += ends[-1]
    return got | {"table": table, "free": s["free"], "count": s["state"][:1], "left": s["lens"]}


def _turned(x, cos, sin, case):
    """x with the first `rot` values of each head turned."""
    rot, head = case["rot"], x[..., :case["rot"]].float()
    a, b = (head[..., :rot // 2], head[..., rot // 2:]) if case["layout"] == "half" else (head[..., ::2], head[..., 1::2])
    a, b = a * cos - b * sin, b * cos + a * sin
    head = torch.cat([a, b], -1) if case["layout"] == "half" else torch.stack([a, b], -1).flatten(-2)
    return torch.cat([head.to(x.dtype), x[..., rot:]], -1)


def _plain_rope(s):
    angle = s["positions"].double()[:, None, None] * s["freq"]
    cos, sin = (torch.cos(angle) * s["factor"]).float(), (torch.sin(angle) * s["factor"]).float()
    return {name: _turned(s[name], cos, sin, s["case"]) for name in ("q", "k")}


def run(s):
    kind = s["case"]["kind"]
    if not own:
        return {"rows": _plain_rows, "attend": _plain_attend, "pages": _plain_pages, "rope": _plain_rope}[kind](s)
    if kind == "rope":
        q, k = s["rope"]((s["q"], s["k"]), s["positions"])
        return {"q": q, "k": k}
    if kind == "pages":
        got = s["pages"].grow(s["counts"], s["rows"], s["names"])
        s["pages"].shrink(s["before"], s["names"])
        return {"slots": got.slots, "positions": got.positions, "starts": got.starts, "lens": got.lens, "pages": got.pages, "table": s["table"],
                "free": s["free"], "count": s["state"][:1], "left": s["lens"]}
    cache = s["cache"]
    if kind == "rows":
        cache.write(s["new_k"], s["new_v"], s["slots"])
        k, v = cache.read(s["slots"])
        return {"k": k, "v": v}
    if not s["case"]["lse"]:
        got = {"out": cache.attend(s["q"], s["pages"], s["lens"], k=s["new_k"], v=s["new_v"])}
    else:
        out, lse = cache.attend(s["q"], s["pages"], s["lens"], k=s["new_k"], v=s["new_v"], lse=True)
        got = {"out": out, "lse": lse}
    if s["new_k"] is not None:
        got["k"], got["v"] = cache.read(s["slots"])
    return got


# ------------------------------------------------------------------ 64 bits, from the definitions
def _kept(x):
    """What is kept of rows x, in 64 bits: sixteen values from the least to the largest one, the distance between them held in bf16."""
    x = x.double()
    least, most = x.min(-1, keepdim=True).values, x.max(-1, keepdim=True).values
    unit = ((most - least) / 15.0).to(torch.bfloat16).double()
    return least + torch.where(unit > 0, torch.round((x - least) / unit), 0.0) * unit


def _exact_rows(case, s):
    return {"k": _kept(s["new_k"]), "v": _kept(s["new_v"])}


def _exact_attend(case, s):
    group = case["heads"] // case["kv_heads"]
    out = torch.zeros(case["batch"], case["heads"], D, dtype=torch.float64, device="cuda")
    lse = torch.full((case["batch"], case["heads"]), -math.inf, dtype=torch.float64, device="cuda")
    for b, n in enumerate(_lens(case)):
        if n == 0:
            continue
        rows, mine = {}, s["pages"][b, :-(-n // case["page"])].long()
        for name in ("k", "v"):
            codes, scales = s[name][mine].short(), s[name + "_scale"][mine].double()
            x = torch.empty(*codes.shape[:3], D, dtype=torch.float64, device="cuda")
            x[..., 0::2], x[..., 1::2] = (codes % 16).double(), torch.div(codes, 16, rounding_mode="floor").double()
            x = (x * scales[..., 0, None] + scales[..., 1, None]).transpose(0, 1).reshape(case["kv_heads"], -1, D)[:, :n]
            if case["append"]:
                x[:, n - 1] = _kept(s["new_" + name][b])
            rows[name] = x
        for h in range(case["heads"]):
            z = torch.mv(rows["k"][h // group], s["q"][b, h].double()) / math.sqrt(D)
            lse[b, h] = torch.logsumexp(z, 0)
            out[b, h] = torch.mv(rows["v"][h // group].T, torch.exp(z - lse[b, h]))
    got = {"out": out}
    if case["lse"]:
        got["lse"] = lse
    return got | (_exact_rows(case, s) if case["append"] else {})


def _exact_rope(case, s):
    rot = case["rot"]
    first = torch.arange(rot // 2, device="cuda") * (1 if case["layout"] == "half" else 2)
    second = first + (rot // 2 if case["layout"] == "half" else 1)
    turn = torch.polar(torch.full((), s["factor"], dtype=torch.float64, device="cuda"), s["positions"].double()[:, None] * s["freq"][None, :])[:, None, :]
    got = {}
    for name in ("q", "k"):
        x = s[name].double().clone()
        z = torch.complex(x[..., first], x[..., second]) * turn
        x[..., first], x[..., second] = z.real, z.imag
        got[name] = x
    return got


def exact(case, seed):
    if case["kind"] == "pages" or (case["kind"] == "attend" and case["batch"] * case["heads"] > 8192):
        return None
    s = prepare(case, seed)
    return {"rows": _exact_rows, "attend": _exact_attend, "rope": _exact_rope}[case["kind"]](case, s)
