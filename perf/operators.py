"""What the performance of the single-row path is measured on: the operators that run a decoder block for the next row of
one or many sequences over keys and values of earlier rows, each in a plain form (elementary torch operations in 32
bits) and through the framework's entry points.

Kinds of case
  cache    KvCache.write, KvCache.read: rows of keys and values into a paged cache (bf16, or quantised as they are
           written: fp8 e4m3 or int8 codes with one fp32 scale for each token and head), and the same rows read back
  attend   KvCache.attend: attention of one new row per sequence over its cached rows, where asked with the new row's key and
           value appended first
  norms    residual_norm: the norm behind a branch, its gate and scale, the residual sum and the next branch's norm
"""
import math

import torch

own = False  # False: the plain forms; True: the framework's operators

D = 128  # width of a head
HIDDEN, HEADS, KV_HEADS, MLP, TOWER = 4096, 32, 8, 12288, 1152
QUANT_MAX = {"int8": 127.0, "fp8": 448.0}
CODES = {"bf16": torch.bfloat16, "fp8": torch.float8_e4m3fn, "int8": torch.int8}
FLOOR = 2.0 ** -100  # the least maximum a scale is made of
EPS = 1e-6


def listed():
    return [
        # the key and value rows of one short prompt, quantised: the smallest write, bound by latency
        {"name": "cache_prompt_77", "kind": "cache", "rows": 77, "kv_heads": 8, "type": "int8", "page": 16, "used": 0.5},
        # a batch of prompts written together: an odd number of rows, scattered over the pages
        {"name": "cache_batch_4111", "kind": "cache", "rows": 4111, "kv_heads": 8, "type": "fp8", "page": 32, "used": 0.8},
        # the rows of the largest sequence the framework is measured on
        {"name": "cache_long_16640", "kind": "cache", "rows": 16640, "kv_heads": 8, "type": "int8", "page": 64, "used": 0.9},
        # one short prompt continued by a row, which is appended by the same call: latency only
        {"name": "attend_one_85", "kind": "attend", "batch": 1, "heads": 32, "kv_heads": 8, "least": 85, "most": 85, "type": "bf16",
         "page": 16, "append": True, "lse": False},
        # a served batch of ragged lengths, the new rows appended
        {"name": "attend_batch_24", "kind": "attend", "batch": 24, "heads": 32, "kv_heads": 8, "least": 1, "most": 2100, "type": "bf16",
         "page": 16, "append": True, "lse": False},
        # one very long sequence: few (sequence, head) pairs, so the length has to be split over the whole GPU
        {"name": "attend_long_100003", "kind": "attend", "batch": 1, "heads": 32, "kv_heads": 8, "least": 100003, "most": 100003,
         "type": "int8", "page": 64, "append": False, "lse": True},
        # a key head for every query head, odd lengths, some sequences empty; its log-sums join it with another part
        {"name": "attend_mha_9", "kind": "attend", "batch": 9, "heads": 16, "kv_heads": 16, "least": 0, "most": 1999, "type": "fp8",
         "page": 32, "append": False, "lse": True},
        # a full server: many long sequences over a quantised cache, bound by memory alone
        {"name": "attend_server_96", "kind": "attend", "batch": 96, "heads": 32, "kv_heads": 8, "least": 300, "most": 5400, "type": "fp8",
         "page": 64, "append": False, "lse": False},
        # the residual and the next norm of a single row
        {"name": "norms_row", "kind": "norms", "rows": 1, "cols": 4096, "post": False, "gate": 0, "mod": False, "alpha": 1.0},
        # both branches of a guided step of 296 rows, each with its own gate and modulation, a norm behind the branch as well
        {"name": "norms_guided_592", "kind": "norms", "rows": 592, "cols": 4096, "post": True, "gate": 2, "mod": True, "alpha": 0.7},
        # rows of the vision tower's width, an odd number of them
        {"name": "norms_tower_4093", "kind": "norms", "rows": 4093, "cols": 1152, "post": True, "gate": 1, "mod": False, "alpha": 0.5},
        # the largest sequence, residual and norm as in the decoder's blocks
        {"name": "norms_16640", "kind": "norms", "rows": 16640, "cols": 4096, "post": False, "gate": 1, "mod": True, "alpha": 1.0},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["cache", "attend", "attend", "attend", "norms"])
    if kind == "cache":
        heads = rng.choice([1, 2, 4, 8, 8, 16])
        return {"kind": kind, "rows": _log(rng, 1, 16640 * 8 // max(8, heads)), "kv_heads": heads, "type": rng.choice(["bf16", "fp8", "int8"]),
                "page": rng.choice([16, 32, 64, 128]), "used": round(rng.uniform(0.3, 0.95), 2)}
    if kind == "attend":
        kv_heads = rng.choice([1, 2, 4, 8, 8, 16])
        heads = kv_heads * rng.choice([1, 2, 3, 4, 4, 7, 8, 16][: 8 if kv_heads <= 4 else 7])
        batch = _log(rng, 1, 128)
        type_ = rng.choice(["bf16", "fp8", "int8"])
        most = _log(rng, 1, min(100003, (1000000 if type_ == "bf16" else 2000000) // (batch * kv_heads)))
        append = type_ == "bf16" and rng.random() < 0.5
        least = rng.choice([most, max(1, most // 2), 1, 0])
        return {"kind": kind, "batch": batch, "heads": heads, "kv_heads": kv_heads, "least": max(1, least) if append else least, "most": most,
                "type": type_, "page": rng.choice([16, 32, 64, 128]), "append": append, "lse": rng.random() < 0.5}
    cols = rng.choice([HIDDEN, HIDDEN, TOWER, _log(rng, 64, MLP), 8 * _log(rng, 16, MLP // 8)])
    rows = _log(rng, 1, 16640 * HIDDEN // max(cols, HIDDEN))
    groups = rng.choice([n for n in (0, 1, 1, 2, 3) if n == 0 or rows % n == 0])
    return {"kind": kind, "rows": rows, "cols": cols, "post": rng.random() < 0.5, "gate": groups, "mod": rng.random() < 0.5,
            "alpha": rng.choice([1.0, 1.0, 0.5, 0.22])}


# ------------------------------------------------------------------ sizes
def _lens(case):
    """Rows of each sequence, the new one included, between least and most."""
    a, b = case["least"], case["most"]
    return [a + int((0.5 + 0.6180339887498949 * i) % 1.0 * (b - a + 1)) for i in range(case["batch"])]


def _row_bytes(case):
    """Bytes of a token's keys and values in the cache."""
    return 2 * case["kv_heads"] * (2 * D if case["type"] == "bf16" else D + 4)


def work(case):
    if case["kind"] == "cache":
        # rows in, codes and scales out, codes and scales in, rows out; the slots twice
        io = case["rows"] * 2 * case["kv_heads"] * D * 2
        return {"bytes": 2 * io + 2 * case["rows"] * _row_bytes(case) + 16 * case["rows"], "flops": 0}
    if case["kind"] == "attend":
        total, new = sum(_lens(case)), case["batch"] * _row_bytes(case) if case["append"] else 0
        io = case["batch"] * case["heads"] * (2 * D * 2 + (4 if case["lse"] else 0))
        tables = 4 * sum(-(-n // case["page"]) + 1 for n in _lens(case))
        return {"bytes": total * _row_bytes(case) + new + io + tables, "flops": 4 * D * case["heads"] * total}
    n = case["rows"] * case["cols"]
    vectors = 2 * case["cols"] * (1 + case["post"] + case["gate"] + 2 * case["mod"] * max(1, case["gate"]))
    return {"bytes": 8 * n + vectors, "flops": n * (9 + 4 * case["post"] + 2 * case["mod"])}


# ------------------------------------------------------------------ inputs
def _gen(seed, salt=0):
    g = torch.Generator(device="cuda")
    g.manual_seed(int(seed) * 131 + salt)
    return g


def _normal(shape, g, std=1.0, mean=0.0):
    return torch.empty(shape, dtype=torch.bfloat16, device="cuda").normal_(mean, std, generator=g)


def _quantised(x, type_):
    """Codes and scales of rows x [..., D]."""
    if type_ == "bf16":
        return x, None
    top = x.float().abs().amax(-1).clamp_min(FLOOR)
    c = x.float() * (QUANT_MAX[type_] / top)[..., None]
    c = c.round().to(torch.int8) if type_ == "int8" else c.to(torch.float8_e4m3fn)
    return c, top / QUANT_MAX[type_]


def _cache(case, pages, g, filled):
    """A cache of so many pages; filled: with keys that have a few strong channels, as projected keys have, and plain values."""
    shape = (pages, case["kv_heads"], case["page"], D)
    s = {}
    for name in ("k", "v"):
        s[name] = torch.zeros(shape, dtype=torch.uint8 if case["type"] == "fp8" else CODES[case["type"]], device="cuda").view(CODES[case["type"]])
        s[name + "_scale"] = None if case["type"] == "bf16" else torch.zeros(shape[:3], device="cuda")
        if not filled:
            continue
        strong = torch.ones(D, dtype=torch.bfloat16, device="cuda")
        if name == "k":
            strong[::17] = 4.0
        step = max(1, (1 << 26) // (shape[1] * shape[2] * D))
        for at in range(0, pages, step):
            c, scale = _quantised(_normal((min(step, pages - at),) + shape[1:], g) * strong, case["type"])
            s[name].view(torch.uint8)[at:at + step] = c.view(torch.uint8)
            if scale is not None:
                s[name + "_scale"][at:at + step] = scale
    return s


def prepare(case, seed):
    g = _gen(seed)
    s = {"case": case}
    if own:
        from __graft_entry__ import load_package
        o1 = load_package()
        o1.use_torch_stream()
        s["o1"] = o1
    if case["kind"] == "norms":
        rows, cols, groups = case["rows"], case["cols"], max(1, case["gate"])
        s["x"], s["branch"] = _normal((rows, cols), g, 2.0), _normal((rows, cols), g, 0.8)
        s["pre"] = _normal((cols,), g, 0.1, 1.0)
        s["post"] = _normal((cols,), g, 0.1, 1.0) if case["post"] else None
        s["gate"] = _normal((groups, cols), g, 0.5) if case["gate"] else None
        s["scale"], s["shift"] = (_normal((groups, cols), g, 0.2), _normal((groups, cols), g, 0.2)) if case["mod"] else (None, None)
        return s
    if case["kind"] == "cache":
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
    if own:
        s["cache"] = s["o1"].KvCache.over(s["k"], s["v"], s["k_scale"], s["v_scale"])
    return s


# ------------------------------------------------------------------ plain forms
def _store(s, slots, new_k, new_v):
    case = s["case"]
    page, at = slots // case["page"], slots % case["page"]
    for name, x in (("k", new_k), ("v", new_v)):
        c, scale = _quantised(x, case["type"])
        s[name].view(torch.uint8)[page, :, at] = c.contiguous().view(torch.uint8)
        if scale is not None:
            s[name + "_scale"][page, :, at] = scale


def _plain_cache(s):
    _store(s, s["slots"], s["new_k"], s["new_v"])
    page, at = s["slots"] // s["case"]["page"], s["slots"] % s["case"]["page"]
    got = []
    for name in ("k", "v"):
        c = s[name].view(torch.uint8)[page, :, at].view(s[name].dtype).float()
        got.append((c if s[name + "_scale"] is None else c * s[name + "_scale"][page, :, at][..., None]).to(torch.bfloat16))
    return {"k": got[0], "v": got[1]}


def _gathered(s, name, table, valid):
    """Rows [batch, kv_heads, width * page, D] in 32 bits, zeros where a sequence has none."""
    x = s[name].view(torch.uint8)[table].view(s[name].dtype).float()
    if s[name + "_scale"] is not None:
        x = x * s[name + "_scale"][table][..., None]
    x = x.permute(0, 2, 1, 3, 4).reshape(table.shape[0], s[name].shape[1], -1, D)
    return x.masked_fill_(~valid[:, None, :, None], 0.0)


def _plain_attend(s):
    case, lens = s["case"], s["lens"].long()
    table = s["pages"].long().clamp_min(0)
    if s["new_k"] is not None:
        last = lens - 1
        page = table.gather(1, (last // case["page"])[:, None])[:, 0]
        _store(s, page * case["page"] + last % case["page"], s["new_k"], s["new_v"])
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
    if s["new_k"] is not None:
        got["k"], got["v"] = s["k"], s["v"]
    return got


def _rows_of(vectors, rows):
    return vectors.float().repeat_interleave(rows // vectors.shape[0], 0)


def _plain_norms(s):
    rows = s["case"]["rows"]
    x, u = s["x"].float(), s["branch"].float()
    if s["post"] is not None:
        u = u * torch.rsqrt(u.square().mean(-1, keepdim=True) + EPS) * s["post"].float()
    if s["gate"] is not None:
        u = u * _rows_of(s["gate"], rows)
    y = x + s["case"]["alpha"] * u
    h = y * torch.rsqrt(y.square().mean(-1, keepdim=True) + EPS) * s["pre"].float()
    if s["scale"] is not None:
        h = h * (1.0 + _rows_of(s["scale"], rows)) + _rows_of(s["shift"], rows)
    return {"y": y.to(torch.bfloat16), "h": h.to(torch.bfloat16)}


def run(s):
    kind = s["case"]["kind"]
    if not own:
        return {"cache": _plain_cache, "attend": _plain_attend, "norms": _plain_norms}[kind](s)
    if kind == "norms":
        y, h = s["o1"].residual_norm(s["x"], s["branch"], s["pre"], post_w=s["post"], gate=s["gate"], scale=s["scale"], shift=s["shift"],
                                     alpha=s["case"]["alpha"], eps=EPS)
        return {"y": y, "h": h}
    cache = s["cache"]
    if kind == "cache":
        cache.write(s["new_k"], s["new_v"], s["slots"])
        k, v = cache.read(s["slots"])
        return {"k": k, "v": v}
    if not s["case"]["lse"]:
        got = {"out": cache.attend(s["q"], s["pages"], s["lens"], k=s["new_k"], v=s["new_v"])}
    else:
        out, lse = cache.attend(s["q"], s["pages"], s["lens"], k=s["new_k"], v=s["new_v"], lse=True)
        got = {"out": out, "lse": lse}
    if s["new_k"] is not None:
        got["k"], got["v"] = s["k"], s["v"]
    return got


# ------------------------------------------------------------------ 64 bits, from the definitions
def _e4m3_64(x):
    """The nearest value of four exponent and three mantissa bits, ties to the even one, at most 448."""
    step = torch.exp2(torch.floor(torch.log2(x.abs().clamp_min(2.0 ** -6))) - 3.0)
    return (torch.round(x / step) * step).clamp(-448.0, 448.0)


def _exact_cache(case, s):
    got = {}
    for name in ("k", "v"):
        x = s["new_" + name].double()
        if case["type"] != "bf16":
            unit = x.abs().amax(-1, keepdim=True).clamp_min(FLOOR) / QUANT_MAX[case["type"]]
            x = (torch.round(x / unit) if case["type"] == "int8" else _e4m3_64(x / unit)) * unit
        got[name] = x
    return got


def _exact_attend(case, s):
    group, page = case["heads"] // case["kv_heads"], case["page"]
    out = torch.zeros(case["batch"], case["heads"], D, dtype=torch.float64, device="cuda")
    lse = torch.full((case["batch"], case["heads"]), -math.inf, dtype=torch.float64, device="cuda")
    for b, n in enumerate(_lens(case)):
        rows = {}
        mine = s["pages"][b, :-(-n // page)].long()
        if n == 0:
            continue
        for name in ("k", "v"):
            x = s[name].view(torch.uint8)[mine].view(s[name].dtype).double()
            if s[name + "_scale"] is not None:
                x *= s[name + "_scale"][mine].double().unsqueeze(-1)
            x = x.transpose(0, 1).reshape(case["kv_heads"], -1, D)[:, :n]
            if case["append"]:
                x[:, n - 1] = s["new_" + name][b].double()
                s[name][mine[-1], :, (n - 1) % page] = s["new_" + name][b]
            rows[name] = x
        for h in range(case["heads"]):
            z = torch.mv(rows["k"][h // group], s["q"][b, h].double()) / math.sqrt(D)
            lse[b, h] = torch.logsumexp(z, 0)
            out[b, h] = torch.mv(rows["v"][h // group].T, torch.exp(z - lse[b, h]))
    got = {"out": out}
    if case["lse"]:
        got["lse"] = lse
    if case["append"]:
        got["k"], got["v"] = s["k"].double(), s["v"].double()
    return got


def _exact_norms(case, s):
    def norm(a, w):
        return a / torch.sqrt((a * a).sum(1, keepdim=True) / a.shape[1] + EPS) * w.double()

    def each(a):
        return a.double().unsqueeze(1).expand(-1, case["rows"] // a.shape[0], -1).reshape(case["rows"], -1)

    branch = s["branch"].double() if s["post"] is None else norm(s["branch"].double(), s["post"])
    y = s["x"].double() + case["alpha"] * (branch if s["gate"] is None else each(s["gate"]) * branch)
    h = norm(y, s["pre"])
    if s["scale"] is not None:
        h = h + h * each(s["scale"]) + each(s["shift"])
    return {"y": y, "h": h}


def exact(case, seed):
    if case["kind"] == "attend" and case["batch"] * case["heads"] > 8192:
        return None
    s = prepare(case, seed)
    return {"cache": _exact_cache, "attend": _exact_attend, "norms": _exact_norms}[case["kind"]](case, s)
