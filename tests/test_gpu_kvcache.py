"""Cached keys and values and the attention of new rows over them, against 64-bit arithmetic on the CPU.

Tolerances, from the arithmetic and not from a run: an output is some value within the bound of the 64-bit one, rounded once to
bf16, so it lies between the bound's two ends as rounded.  The bound: a probability has the error of its exponent (q . k summed in fp32:
2^-19 of the sum of its terms' magnitudes, covering any order and a truncating sum) and, where it multiplies v, 2^-12 of itself
(fp8, int8 caches) or 2^-17 (bf16 caches).  All are relative to sum p |v| / l."""
import ctypes as C
import math

import pytest
import torch

D = 128
QMAX = {"int8": 127.0, "fp8": 448.0}
gpu = pytest.mark.gpu


def gen(seed):
    return torch.Generator().manual_seed(seed)


def normal(shape, g, std=1.0):
    return (torch.randn(shape, generator=g) * std).to(torch.bfloat16)


def quantised(x, kind):
    """Codes and scales of bf16 rows by the definition, in fp32 with its roundings."""
    if kind == "bf16":
        return x, None
    q = torch.tensor(QMAX[kind])
    a = x.float().abs().amax(-1).clamp_min(2.0 ** -100)
    good = torch.isfinite(x.float()).all(-1)
    scale = torch.where(good, a / q, math.nan)
    inv = torch.where(good, q / a, 0.0)
    y = torch.where(good[..., None], x.float() * inv[..., None], 0.0)
    return (y.round().to(torch.int8) if kind == "int8" else y.to(torch.float8_e4m3fn)), scale


def value(codes, scale):
    return codes.float().double() if scale is None else codes.float().double() * scale.double()[..., None]


def between(got, ref, tol, what=""):
    """got is a value within tol of ref, rounded to bf16."""
    got = got.cpu().double()
    ok = (got >= (ref - tol).to(torch.bfloat16).double()) & (got <= (ref + tol).to(torch.bfloat16).double())
    assert ok.all(), f"{what}: {int((~ok).sum())} of {ok.numel()} outside; the worst {((got - ref).abs() / tol)[~ok].max():.3g} times the bound from 64 bits"


class Case:
    """A cache with rows of known values at random pages, everything else in it unusable: NaN and Inf where the type has them."""

    def __init__(self, o1, dev, kind, lens, kv_heads, page, seed=0, std=1.0, width_extra=2, table_junk=True):
        g = gen(seed)
        self.kind, self.lens, self.hk, self.page = kind, lens, kv_heads, page
        need = [-(-n // page) for n in lens]
        pages = sum(need) + 2
        order = torch.randperm(pages, generator=g)
        self.table = torch.full((len(lens), max(need + [1]) + width_extra), 2 ** 30 if table_junk else 0, dtype=torch.int32)
        at = 0
        for b, n in enumerate(need):
            self.table[b, :n] = order[at:at + n].int()
            at += n
        self.k = [normal((n, kv_heads, D), g, std) for n in lens]
        self.v = [normal((n, kv_heads, D), g) for n in lens]
        self.cache = o1.KvCache(pages, page, kind, kv_heads, dev)
        for t in (self.cache.k, self.cache.v):
            if kind == "bf16":
                t.view(torch.int16).random_(-32768, 32767)
                t.view(torch.int16)[:, :, ::3] = 0x7FC0      # NaN
                t.view(torch.int16)[:, :, 1::3] = 0x7F80     # Inf
            elif kind == "fp8":
                t.view(torch.uint8).fill_(0x7F)              # NaN
            else:
                t.fill_(127)
        for t in (self.cache.k_scale, self.cache.v_scale):
            if t is not None:
                t.fill_(math.nan)
                t[:, :, ::2] = math.inf
        self.dev = dev
        self.dtable, self.dlens = self.table.to(dev), torch.tensor(lens, dtype=torch.int32, device=dev)

    def slots(self, b, lo=0, hi=None):
        t = torch.arange(lo, self.lens[b] if hi is None else hi)
        return (self.table[b].long()[t // self.page] * self.page + t % self.page)

    def fill(self, but_last=False):
        """All rows written in one call, in an order of their own."""
        cut = [max(0, n - 1) if but_last else n for n in self.lens]
        if not sum(cut):
            return
        k = torch.cat([x[:n] for x, n in zip(self.k, cut)])
        v = torch.cat([x[:n] for x, n in zip(self.v, cut)])
        s = torch.cat([self.slots(b, 0, n) for b, n in enumerate(cut)])
        p = torch.randperm(len(s), generator=gen(5))
        self.cache.write(k[p].contiguous().to(self.dev), v[p].contiguous().to(self.dev), s[p].to(self.dev))

    def reference(self, q, scale=None):
        """out, lse and the bounds of both, in 64 bits from the definition."""
        B, H = q.shape[:2]
        G = H // self.hk
        sc = D ** -0.5 if scale is None else scale
        out, lse = torch.zeros(B, H, D, dtype=torch.float64), torch.full((B, H), -math.inf, dtype=torch.float64)
        tol_o, tol_l = torch.zeros_like(out), torch.zeros_like(lse)
        for b, n in enumerate(self.lens):
            if n == 0:
                continue
            k, v = (value(*quantised(x[b], self.kind)).repeat_interleave(G, 1) for x in (self.k, self.v))
            qd = q[b].double()
            z = torch.einsum("hd,thd->ht", qd, k) * sc
            size = (torch.einsum("hd,thd->ht", qd.abs(), k.abs()) * sc).amax(-1)
            lse[b] = torch.logsumexp(z, -1)
            p = torch.exp(z - lse[b][:, None])
            out[b] = torch.einsum("ht,thd->hd", p, v)
            spread = torch.einsum("ht,thd->hd", p, v.abs())
            rel = 2.0 * 2.0 ** -19 * size + (2.0 ** -17 if self.kind == "bf16" else 2.0 ** -12) + 2.0 ** -18
            tol_o[b] = spread * rel[:, None] + 1e-30
            tol_l[b] = 2.0 ** -19 * size + 2.0 ** -21 * (1 + lse[b].abs())
        return out, lse, tol_o, tol_l

    def check(self, q, got, lse=None, scale=None, what=""):
        ref, ref_l, tol_o, tol_l = self.reference(q, scale)
        assert torch.isfinite(got.float()).all(), f"{what}: not finite"
        between(got, ref, tol_o, what)
        if lse is not None:
            empty = torch.tensor(self.lens) == 0
            assert (lse.cpu()[empty] == -math.inf).all()
            d = (lse.cpu().double() - ref_l).abs()[~empty]
            assert (d <= tol_l[~empty]).all(), f"{what}: lse off by {(d / tol_l[~empty]).max():.3g} times the bound"


# ------------------------------------------------------------------ write and read
@gpu
@pytest.mark.parametrize("kind", ["bf16", "fp8", "int8"])
@pytest.mark.parametrize("rows,heads,page", [(1, 1, 16), (1, 8, 64), (37, 8, 48), (515, 3, 16), (64, 16, 128)])
def test_rows_written_and_read_back(pkg, dev, kind, rows, heads, page):
    g = gen(rows + heads)
    pages = -(-rows // page) + 3
    cache = pkg.KvCache(pages, page, kind, heads, dev)
    k, v = normal((rows, heads, D), g, 2.0), normal((rows, heads, D), g)
    k[:, :, ::13] *= 50
    if rows > 3:
        k[0], v[1], k[2, 0] = 0.0, 2.0 ** -130, -0.0
        v[3] = 2.0 ** 120
        k[1, 0, 5], v[2, heads - 1, 7], v[3, 0, 0] = math.nan, math.inf, -math.inf
    slots = torch.randperm(pages * page, generator=g)[:rows]
    cache.write(k.to(dev), v.to(dev), slots.to(dev))
    got = cache.read(slots.to(dev))
    torch.cuda.synchronize()
    for name, x, y, store, scales in (("k", k, got[0], cache.k, cache.k_scale), ("v", v, got[1], cache.v, cache.v_scale)):
        codes, scale = quantised(x, kind)
        page_at, at = slots // page, slots % page
        held = store.cpu().view(torch.uint8 if kind != "bf16" else torch.int16)[page_at, :, at]
        assert torch.equal(held, codes.view(held.dtype)), name + ": codes"
        want = x
        if kind != "bf16":
            s = scales.cpu()[page_at, :, at]
            assert torch.equal(torch.isnan(s), torch.isnan(scale)) and torch.equal(s.nan_to_num(0), scale.nan_to_num(0)), name + ": scales"
            want = (codes.float() * scale[..., None]).to(torch.bfloat16)
        y = y.cpu()
        assert torch.equal(torch.isnan(y), torch.isnan(want)) and torch.equal(y.nan_to_num(7), want.nan_to_num(7)), name + ": read back"
    # what was not written is as it was
    mask = torch.ones(pages * page, dtype=torch.bool)
    mask[slots] = False
    rest = cache.k.cpu().view(torch.uint8).permute(0, 2, 1, 3).reshape(pages * page, -1)[mask]
    assert (rest == 0).all()


@gpu
@pytest.mark.parametrize("kind", ["bf16", "fp8", "int8"])
@pytest.mark.parametrize("off,pad", [(0, 0), (0, 64), (1, 0), (8, 8), (3, 5)])
def test_rows_of_other_pitches_and_alignments(pkg, dev, kind, off, pad):
    """Rows inside wider ones (q | k | v), at addresses of 2 bytes, give the codes that rows by themselves give."""
    g, rows, heads = gen(3), 29, 4
    k, v = normal((rows, heads, D), g), normal((rows, heads, D), g)
    slots = torch.randperm(64, generator=g)[:rows].to(dev)
    a, b = pkg.KvCache(4, 16, kind, heads, dev), pkg.KvCache(4, 16, kind, heads, dev)
    a.write(k.to(dev), v.to(dev), slots)
    wide = torch.zeros(rows * (2 * heads * D + pad) + off, dtype=torch.bfloat16, device=dev)
    w = wide[off:].view(rows, -1)
    w[:, :heads * D], w[:, heads * D:2 * heads * D] = k.to(dev).view(rows, -1), v.to(dev).view(rows, -1)
    wk, wv = (w[:, i * heads * D:(i + 1) * heads * D].unflatten(1, (heads, D)) for i in (0, 1))
    b.write(wk, wv, slots)
    assert torch.equal(a.k.view(torch.uint8), b.k.view(torch.uint8)) and torch.equal(a.v.view(torch.uint8), b.v.view(torch.uint8))
    want = a.read(slots)
    wide.fill_(7.0)
    a.read(slots, out=(wk, wv))
    assert torch.equal(wk, want[0]) and torch.equal(wv, want[1])
    if pad:
        assert (w[:, 2 * heads * D:] == 7.0).all()
    assert (wide[:off] == 7.0).all()


@gpu
def test_negative_and_wrong_slots(pkg, dev):
    cache = pkg.KvCache(2, 16, "int8", 2, dev)
    x = normal((4, 2, D), gen(1)).to(dev)
    cache.write(x, x, torch.tensor([-1, 3, -5, 31], device=dev))
    k, v = cache.read(torch.tensor([3, -2, 31, 0], device=dev))
    assert pkg.lib.o1_device_error() == 0
    assert (k[1] == 0).all() and (v[1] == 0).all() and (k[3] == 0).all() and (k[0] != 0).any()
    before = cache.k.clone()
    cache.write(x, x, torch.tensor([32, -1, -1, 2 ** 40], device=dev))
    assert pkg.lib.o1_device_error() == 70
    assert torch.equal(before, cache.k)
    k, _ = cache.read(torch.tensor([32], device=dev))
    assert (k == 0).all() and pkg.lib.o1_device_error() == 70
    cache.write(x[:0], x[:0], torch.zeros(0, dtype=torch.int64, device=dev))
    assert cache.read(torch.zeros(0, dtype=torch.int64, device=dev))[0].shape == (0, 2, D)


# ------------------------------------------------------------------ attention
LENS = [0, 1, 2, 15, 16, 17, 31, 33, 64, 65, 100, 127, 128, 129, 200, 255, 257, 300]


@gpu
@pytest.mark.parametrize("kind", ["bf16", "fp8", "int8"])
@pytest.mark.parametrize("kv_heads,group,page", [(8, 4, 16), (1, 1, 16), (2, 8, 64), (3, 3, 48), (2, 7, 32), (1, 16, 128), (2, 12, 16), (1, 24, 64),
                                                 (1, 33, 16), (16, 1, 32)])
def test_attention_of_ragged_sequences(pkg, dev, kind, kv_heads, group, page):
    c = Case(pkg, dev, kind, LENS, kv_heads, page, seed=kv_heads * 100 + group)
    c.fill()
    q = normal((len(LENS), kv_heads * group, D), gen(9), 2.0)
    out, lse = c.cache.attend(q.to(dev), c.dtable, c.dlens, lse=True)
    c.check(q, out, lse, what=kind)
    again, lse2 = c.cache.attend(q.to(dev), c.dtable, c.dlens, lse=True)
    assert torch.equal(out, again) and torch.equal(lse, lse2)
    assert torch.equal(out, c.cache.attend(q.to(dev), c.dtable, c.dlens))


@gpu
@pytest.mark.parametrize("kind", ["bf16", "fp8", "int8"])
@pytest.mark.parametrize("lens,kv_heads,group", [([1], 1, 1), ([1], 8, 4), ([85], 8, 4), ([4097], 8, 4), ([30011], 1, 8), ([30011], 2, 16), ([9001, 1, 0, 12000, 3], 2, 4),
                                                 ([700] * 40, 1, 4), ([0, 0, 0], 2, 2), ([257] * 300, 1, 2), ([1] * 700 + [5000], 1, 1)])
def test_attention_over_few_and_many_rows(pkg, dev, kind, lens, kv_heads, group):
    """One long sequence (split and joined), many short ones, both beside each other."""
    c = Case(pkg, dev, kind, lens, kv_heads, 32, seed=len(lens))
    c.fill()
    q = normal((len(lens), kv_heads * group, D), gen(11), 1.5)
    out, lse = c.cache.attend(q.to(dev), c.dtable, c.dlens, lse=True)
    c.check(q, out, lse, what=kind)
    for _ in range(3):
        again, lse2 = c.cache.attend(q.to(dev), c.dtable, c.dlens, lse=True)
        assert torch.equal(out, again) and torch.equal(lse, lse2)


@gpu
@pytest.mark.parametrize("kind", ["bf16", "fp8", "int8"])
@pytest.mark.parametrize("lens,kv_heads,group,page", [([1, 16, 17, 0, 33, 128, 2, 129], 8, 4, 16), ([1], 8, 4, 64), ([20000], 2, 4, 64), ([5, 700, 1300], 1, 24, 48),
                                                      ([3] * 90, 4, 1, 16)])
def test_new_rows_appended_by_the_same_call(pkg, dev, kind, lens, kv_heads, group, page):
    """As write and then attend: the same cache afterwards, and the same bits."""
    a, b = (Case(pkg, dev, kind, lens, kv_heads, page, seed=4) for _ in range(2))
    a.fill()
    b.cache.k.copy_(a.cache.k)
    b.cache.v.copy_(a.cache.v)
    for n in ("k_scale", "v_scale"):
        if getattr(a.cache, n) is not None:
            getattr(b.cache, n).copy_(getattr(a.cache, n))
    last = [b.slots(i)[-1] for i, n in enumerate(lens) if n]
    for t in (b.cache.k.view(torch.uint8), b.cache.v.view(torch.uint8)):
        for s in last:
            t[int(s) // page, :, int(s) % page] = 0x7F      # a stale row where the new one goes
    new = torch.zeros(len(lens), 2 * kv_heads * D, dtype=torch.bfloat16)
    for i, n in enumerate(lens):
        if n:
            new[i, :kv_heads * D], new[i, kv_heads * D:] = b.k[i][-1].flatten(), b.v[i][-1].flatten()
    new = new.to(dev)
    q = normal((len(lens), kv_heads * group, D), gen(12))
    out, lse = b.cache.attend(q.to(dev), b.dtable, b.dlens, k=new[:, :kv_heads * D].unflatten(1, (kv_heads, D)),
                              v=new[:, kv_heads * D:].unflatten(1, (kv_heads, D)), lse=True)
    want, want_l = a.cache.attend(q.to(dev), a.dtable, a.dlens, lse=True)
    assert torch.equal(a.cache.k.view(torch.uint8), b.cache.k.view(torch.uint8))
    assert torch.equal(a.cache.v.view(torch.uint8), b.cache.v.view(torch.uint8))
    if kind != "bf16":
        for n in ("k_scale", "v_scale"):
            assert torch.equal(getattr(a.cache, n).view(torch.int32), getattr(b.cache, n).view(torch.int32))
    assert torch.equal(out, want) and torch.equal(lse, want_l)
    b.check(q, out, lse, what=kind)


MANY = [(300, 4, 4, 16, 90), (130, 8, 7, 32, 64), (230, 2, 16, 32, 33), (160, 3, 24, 16, 48), (470, 1, 1, 48, 48), (64, 16, 3, 16, 33), (600, 8, 2, 16, 200)]


@gpu
@pytest.mark.parametrize("kind", ["bf16", "fp8", "int8"])
@pytest.mark.parametrize("batch,kv_heads,group,page,most", MANY)
def test_many_short_sequences(pkg, dev, kind, batch, kv_heads, group, page, most):
    """More (sequence, kv head) pairs than the GPU has teams of warps, a short table: a pair to a warp, lengths from 0."""
    lens = [(37 * b) % (most + 1) for b in range(batch)]
    c = Case(pkg, dev, kind, lens, kv_heads, page, seed=batch)
    c.fill()
    q = normal((batch, kv_heads * group, D), gen(13), 1.5)
    out, lse = c.cache.attend(q.to(dev), c.dtable, c.dlens, lse=True)
    assert pkg.lib.o1_device_error() == 0
    c.check(q, out, lse, what=kind)
    again, lse2 = c.cache.attend(q.to(dev), c.dtable, c.dlens, lse=True)
    assert torch.equal(out, again) and torch.equal(lse, lse2)
    # in a wide table the pairs go to teams
    wide = torch.full((batch, 300), -1, dtype=torch.int32, device=dev)
    wide[:, :c.dtable.size(1)] = c.dtable
    out, lse = c.cache.attend(q.to(dev), wide, c.dlens, lse=True)
    c.check(q, out, lse, what=kind)


@gpu
@pytest.mark.parametrize("kind", ["bf16", "fp8", "int8"])
@pytest.mark.parametrize("batch,kv_heads,group,page,most", [(300, 4, 4, 16, 90), (230, 2, 16, 32, 33), (470, 1, 1, 48, 48)])
def test_many_short_sequences_with_new_rows(pkg, dev, kind, batch, kv_heads, group, page, most):
    test_new_rows_appended_by_the_same_call(pkg, dev, kind, [(37 * b) % (most + 1) for b in range(batch)], kv_heads, group, page)


@gpu
def test_many_short_sequences_with_wrong_tables(pkg, dev):
    lens = [1 + b % 40 for b in range(260)]
    c = Case(pkg, dev, "fp8", lens, 2, 16)
    c.fill()
    q = normal((260, 8, D), gen(1)).to(dev)
    good = c.cache.attend(q, c.dtable, c.dlens)
    assert pkg.lib.o1_device_error() == 0
    t, ln = c.dtable.clone(), c.dlens.clone()
    t[100, 0], t[7, 0] = c.cache.pages, -1
    out = c.cache.attend(q, t, c.dlens)
    rest = [b for b in range(260) if b not in (7, 100)]
    assert pkg.lib.o1_device_error() == 70 and torch.equal(out[rest], good[rest])
    ln[100], ln[7] = -1, 16 * c.table.shape[1] + 1
    out = c.cache.attend(q, c.dtable, ln)
    assert pkg.lib.o1_device_error() == 71 and torch.equal(out[rest], good[rest])


@gpu
@pytest.mark.parametrize("kind", ["bf16", "fp8", "int8"])
def test_scores_of_any_size(pkg, dev, kind):
    """Scores of thousands (one key takes all), rows that rise and fall, keys of different magnitudes, tiny and huge values and queries."""
    lens = [300, 1000, 77, 513]
    c = Case(pkg, dev, kind, lens, 2, 16, seed=7, std=30.0)
    ramp = torch.linspace(0.01, 3, 1000)[:, None, None]
    c.k[1], c.k[3] = (c.k[1].float() * ramp).to(torch.bfloat16), (c.k[3].float() * ramp.flip(0)[:513]).to(torch.bfloat16)
    c.v[0], c.v[2] = c.v[0] * 2.0 ** -60, c.v[2] * 2.0 ** 60
    c.v[1] = (c.v[1].float() * torch.logspace(-6, 6, 1000)[:, None, None]).to(torch.bfloat16)
    c.fill()
    q = normal((4, 8, D), gen(3), 4.0)
    q[1, 1], q[2, 2], q[0, 3], q[3, 0] = q[1, 1] * 2.0 ** -70, 0.0, q[0, 3] * 1000, q[3, 0] * 2.0 ** -14
    out, lse = c.cache.attend(q.to(dev), c.dtable, c.dlens, lse=True)
    c.check(q, out, lse, what=kind)
    out, lse = c.cache.attend(q.to(dev), c.dtable, c.dlens, lse=True, scale=0.5)
    c.check(q, out, lse, scale=0.5, what=kind)


@gpu
@pytest.mark.parametrize("kind", ["bf16", "fp8", "int8"])
def test_not_finite_rows_stay_where_they_are(pkg, dev, kind):
    """A NaN in a cached row reaches the sequences that have the row, and no other."""
    lens = [40, 40, 700, 700]
    c = Case(pkg, dev, kind, lens, 1, 16, seed=2)
    c.k[1][20, 0, 3], c.v[3][600, 0, 5] = math.nan, math.nan
    c.fill()
    q = normal((4, 4, D), gen(3)).to(dev)
    out, lse = c.cache.attend(q, c.dtable, c.dlens, lse=True)
    assert torch.isfinite(out[0]).all() and torch.isfinite(out[2]).all() and torch.isfinite(lse[[0, 2, 3]]).all()
    assert torch.isnan(out[1]).all() and torch.isnan(lse[1]).all()
    bad = torch.isnan(out[3])
    assert bad[:, 5].all() and (bad.all() if kind != "bf16" else bad.sum() == 4)


@gpu
def test_pitches_of_queries_and_results(pkg, dev):
    lens, hk, H = [5, 60, 129], 2, 6
    c = Case(pkg, dev, "bf16", lens, hk, 16)
    c.fill()
    q = normal((3, H, D), gen(1))
    want, lse = c.cache.attend(q.to(dev), c.dtable, c.dlens, lse=True)
    c.check(q, want, lse)
    for off, pad in ((0, 256), (8, 8), (1, 0), (3, 7)):
        buf = torch.zeros(3 * (H * D + pad) + off, dtype=torch.bfloat16, device=dev)
        view = buf[off:].view(3, -1)[:, :H * D].unflatten(1, (H, D))
        view.copy_(q.to(dev))
        assert torch.equal(want, c.cache.attend(view, c.dtable, c.dlens))
        buf.fill_(5.0)
        got = c.cache.attend(q.to(dev), c.dtable, c.dlens, out=view)
        assert got.data_ptr() == view.data_ptr() and torch.equal(view, want)
        assert (buf[off:].view(3, -1)[:, H * D:] == 5.0).all() and (buf[:off] == 5.0).all()
    wide = torch.full((3, 50), -7, dtype=torch.int32, device=dev)
    wide[:, :c.table.shape[1]] = c.dtable
    assert torch.equal(want, c.cache.attend(q.to(dev), wide[:, :c.table.shape[1]], c.dlens))


@gpu
def test_tables_that_do_not_fit(pkg, dev):
    """A page outside the cache and lengths outside the table are found on the device, and nothing outside is touched."""
    lens = [40, 20, 16]
    c = Case(pkg, dev, "int8", lens, 2, 16)
    c.fill()
    q = normal((3, 4, D), gen(1))
    good = c.cache.attend(q.to(dev), c.dtable, c.dlens)
    assert pkg.lib.o1_device_error() == 0
    for page in (c.cache.pages, -1, 2 ** 31 - 1, -2 ** 31):
        t = c.dtable.clone()
        t[0, 1] = page
        out = c.cache.attend(q.to(dev), t, c.dlens)
        assert pkg.lib.o1_device_error() == 70 and torch.equal(out[1:], good[1:])
    new = normal((3, 2, D), gen(2)).to(dev)
    for n in (-1, 16 * c.table.shape[1] + 1, 2 ** 31 - 1, -2 ** 31):
        ln = c.dlens.clone()
        ln[0] = n
        out = c.cache.attend(q.to(dev), c.dtable, ln)
        assert pkg.lib.o1_device_error() == 71 and torch.equal(out[1:], good[1:])
    before = c.cache.k.clone()
    ln = torch.tensor([-3, 2 ** 30, 0], dtype=torch.int32, device=dev)
    c.cache.attend(q.to(dev), c.dtable, ln, k=new, v=new)
    assert pkg.lib.o1_device_error() == 71 and torch.equal(before, c.cache.k)
    assert torch.equal(good, c.cache.attend(q.to(dev), c.dtable, c.dlens))
    assert pkg.lib.o1_device_error() == 0
    empty = torch.zeros(3, 0, dtype=torch.int32, device=dev)
    assert (c.cache.attend(q.to(dev), empty, torch.zeros(3, dtype=torch.int32, device=dev)) == 0).all()
    assert c.cache.attend(q[:0].to(dev), c.dtable[:0], c.dlens[:0]).shape == (0, 4, D)


@gpu
def test_offsets_past_32_bits(pkg, dev):
    """A cache of more than 2^32 values, with rows at its end."""
    heads, page = 8, 128
    pages = 2 ** 32 // (heads * page * D) + 40
    cache = pkg.KvCache(pages, page, "int8", heads, dev)
    c = Case(pkg, dev, "int8", [300, 128], heads, page, width_extra=0)
    c.cache = cache
    c.table += (pages - 10) - 0
    c.dtable = c.table.to(dev)
    c.table[c.table >= pages] = 0
    c.dtable = c.table.to(dev)
    c.fill()
    k, _ = cache.read(c.slots(0).to(dev))
    assert torch.equal(k.cpu().double(), value(*quantised(c.k[0], "int8")).to(torch.bfloat16).double())
    q = normal((2, 32, D), gen(3))
    c.check(q, c.cache.attend(q.to(dev), c.dtable, c.dlens))


@gpu
def test_other_streams_and_graphs(pkg, dev):
    """Two streams in turn, each with its own workspace, and a captured call that sees new lengths and new rows."""
    lens = [3000, 17, 900]
    c = Case(pkg, dev, "fp8", lens, 4, 32)
    c.fill()
    q = normal((3, 16, D), gen(3)).to(dev)
    want = c.cache.attend(q, c.dtable, c.dlens)
    torch.cuda.synchronize()
    streams, outs = [torch.cuda.Stream() for _ in range(2)], []
    try:
        for _ in range(6):
            for s in streams:
                with torch.cuda.stream(s):
                    pkg.use_torch_stream()
                    outs.append(c.cache.attend(q, c.dtable, c.dlens))
        torch.cuda.synchronize()
        assert all(torch.equal(o, want) for o in outs)
        table, ln, out = c.dtable.clone(), c.dlens.clone(), torch.empty_like(want)
        with torch.cuda.stream(streams[0]):
            pkg.use_torch_stream()
            c.cache.attend(q, table, ln, out=out)
            torch.cuda.synchronize()
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph, stream=streams[0]):
                pkg.use_torch_stream()
                c.cache.attend(q, table, ln, out=out)
                c.cache.attend(q, table, ln, out=out)
        ln.copy_(torch.tensor([100, 0, 33], dtype=torch.int32))
        graph.replay()
        torch.cuda.synchronize()
    finally:
        pkg.use_torch_stream()
    assert torch.equal(out, c.cache.attend(q, c.dtable, torch.tensor([100, 0, 33], dtype=torch.int32, device=dev)))


@gpu
def test_captures_share_no_workspace(pkg, dev):
    """The first call on a stream may be a captured one; graphs of one stream, replayed in any order or on other streams, and calls outside do not share scratch."""
    c = Case(pkg, dev, "int8", [5000, 2000], 1, 32)
    c.fill()
    host = normal((2, 8, D), gen(3))
    q = host.to(dev)
    outs = [torch.zeros(2, 8, D, dtype=torch.bfloat16, device=dev) for _ in range(4)]
    s, other = torch.cuda.Stream(), torch.cuda.Stream()
    try:
        graphs = []
        for i in range(2):
            torch.cuda.synchronize()
            graphs.append(torch.cuda.CUDAGraph())
            with torch.cuda.graph(graphs[i], stream=s):
                pkg.use_torch_stream()
                assert pkg.lib.o1_capture_id() != 0
                c.cache.attend(q, c.dtable, c.dlens, out=outs[i])
                c.cache.attend(q, c.dtable, c.dlens, out=outs[i])
        with torch.cuda.stream(s):
            pkg.use_torch_stream()
            assert pkg.lib.o1_capture_id() == 0
            c.cache.attend(q, c.dtable, c.dlens, out=outs[2])
        assert len(c.cache._work) == 3 and len({t.data_ptr() for t in c.cache._work.values()}) == 3
        torch.cuda.synchronize()
        for _ in range(5):
            with torch.cuda.stream(s):
                graphs[1].replay()
            with torch.cuda.stream(other):
                graphs[0].replay()
        torch.cuda.synchronize()
    finally:
        pkg.use_torch_stream()
    c.cache.attend(q, c.dtable, c.dlens, out=outs[3])
    assert all(torch.equal(o, outs[3]) for o in outs)
    c.check(host, outs[0])


# ------------------------------------------------------------------ refusals
@gpu
def test_arguments_that_do_not_fit(pkg, dev):
    E = pkg.O1Error
    with pytest.raises(E, match="kind"):
        pkg.KvCache(4, 16, "int4", 2, dev)
    with pytest.raises(E, match="multiple of 16"):
        pkg.KvCache(4, 24, "bf16", 2, dev)
    c = pkg.KvCache(4, 16, "int8", 2, dev)
    with pytest.raises(E, match="scales"):
        pkg.KvCache.over(c.k, c.v)
    with pytest.raises(E, match="contiguous"):
        pkg.KvCache.over(c.k.transpose(0, 1), c.v.transpose(0, 1), c.k_scale.transpose(0, 1), c.v_scale.transpose(0, 1))
    with pytest.raises(E, match="differs"):
        pkg.KvCache.over(c.k, c.v[:2], c.k_scale, c.v_scale)
    x, s = normal((3, 2, D), gen(0)).to(dev), torch.arange(3, device=dev)
    for bad in (x.float(), x[:, :1], x[..., :64], x.cpu(), normal((2, 3, D), gen(0)).to(dev).transpose(0, 1)):
        with pytest.raises(E, match="KvCache.write"):
            c.write(bad, x, s)
    with pytest.raises(E, match="slots int64"):
        c.write(x, x, s.int())
    with pytest.raises(E, match="rows"):
        c.write(x, x, s[:2])
    q, pages, lens = normal((3, 4, D), gen(0)).to(dev), torch.zeros(3, 1, dtype=torch.int32, device=dev), torch.ones(3, dtype=torch.int32, device=dev)
    for args in ((q[0], pages, lens), (q, pages.long(), lens), (q, pages[:2], lens), (q, pages, lens.long()), (q, pages, lens[:1])):
        with pytest.raises(E, match="KvCache.attend"):
            c.attend(*args)
    with pytest.raises(E, match="both or neither"):
        c.attend(q, pages, lens, k=x)
    with pytest.raises(E, match="kv_heads"):
        c.attend(normal((3, 3, D), gen(0)).to(dev), pages, lens)
    with pytest.raises(E, match="scale"):
        c.attend(q, pages, lens, scale=0.0)
    with pytest.raises(E, match="lse"):
        c.attend(q, pages, lens, lse=torch.zeros(3, 3, device=dev))
    pkg.check_cuda_errbuf("after refusals")


def test_entry_points_refuse_before_they_touch_the_gpu(pkg):
    lib, K = pkg.lib, pkg.KvCacheC
    one, odd = C.c_void_p(4096), C.c_void_p(4104)
    good = dict(k=4096, v=4096, k_scale=4096, v_scale=4096, type=2, pages=4, page_size=16, kv_heads=2, head_dim=128)

    def write(rows=1, ld=256, slots=one, k=one, **change):
        return lib.o1_kv_write(C.byref(K(**{**good, **change})), k, ld, one, ld, slots, rows)

    for want, args in ((6, dict(k=None)), (6, dict(slots=None)), (9, dict(rows=-1)), (9, dict(ld=255)), (9, dict(type=3)), (9, dict(head_dim=64)), (9, dict(page_size=8)),
                       (9, dict(page_size=0)), (9, dict(pages=0)), (9, dict(kv_heads=0)), (6, dict(k_scale=None)), (9, dict(v_scale=4100))):
        assert write(**args) == want, args
        assert b"kv_write" in lib.hd_cuda_last_error(), args
    assert lib.o1_kv_write(None, one, 256, one, 256, one, 1) == 6
    assert write(rows=0) == 0 and lib.o1_kv_read(C.byref(K(**good)), one, 256, one, 256, one, 0) == 0
    assert lib.o1_kv_read(C.byref(K(**{**good, "v": None})), one, 256, one, 256, one, 1) == 6
    assert lib.o1_kv_read(C.byref(K(**{**good, "k": 4104})), one, 256, one, 256, one, 1) == 9
    need = lib.o1_kv_attention_workspace_bytes(4, 2)

    def attend(q=one, ldq=512, kn=None, ldk=256, vn=None, ldv=256, pages=one, ldp=3, width=3, lens=one, out=one, ldo=512, batch=1, heads=4, scale=0.1,
               ws=one, nb=need, **change):
        return lib.o1_kv_attention(C.byref(K(**{**good, **change})), q, ldq, kn, ldk, vn, ldv, pages, ldp, width, lens, out, ldo, None, batch, heads, scale, ws, nb)

    for want, args in ((6, dict(q=None)), (6, dict(pages=None)), (6, dict(lens=None)), (6, dict(out=None)), (6, dict(ws=None)), (6, dict(kn=one)), (6, dict(vn=one)),
                       (9, dict(heads=3)), (9, dict(heads=0)), (9, dict(batch=-1)), (9, dict(width=-1)), (9, dict(ldq=511)), (9, dict(ldo=8)), (9, dict(ldp=2)),
                       (9, dict(kn=one, vn=one, ldk=255)), (9, dict(scale=0.0)), (9, dict(scale=math.nan)), (9, dict(scale=math.inf)), (9, dict(scale=-1.0)), (7, dict(nb=need - 1)),
                       (7, dict(ws=odd)), (9, dict(head_dim=72))):
        assert attend(**args) == want, args
        assert b"kv_attention" in lib.hd_cuda_last_error(), args
    assert attend(batch=0) == 0
    lib.hd_cuda_clear_error()


def test_tables_and_heads_beyond_32_bits_are_refused(pkg):
    """The stream of chunks and its costs are counted in 32 bits; what does not fit is refused on the host, before anything is launched."""
    K, lib, one = pkg.KvCacheC, pkg.lib, 4096

    def attend(heads=4, width=3, pages=8, kv_heads=2):
        c = K(one, one, None, None, 0, pages, 16, kv_heads, 128)
        need = lib.o1_kv_attention_workspace_bytes(heads, kv_heads)
        return lib.o1_kv_attention(C.byref(c), one, heads * 128, None, 0, None, 0, one, width, width, one, one, heads * 128, None, 1, heads, 0.1, one, need)

    for args in (dict(heads=1 << 24), dict(heads=1 << 23), dict(width=1 << 27), dict(pages=1 << 27), dict(kv_heads=4096, heads=4096, width=1 << 20)):
        assert attend(**args) == 9, args
        assert b"too large" in lib.hd_cuda_last_error(), args
    lib.hd_cuda_clear_error()


@gpu
def test_a_wrong_slot_stops_no_other_call(pkg, dev):
    """A slot outside the cache is reported, and a product enqueued behind it is made all the same."""
    cache = pkg.KvCache(2, 16, "int8", 2, dev)
    x = normal((1, 2, D), gen(1)).to(dev)
    a, w = normal((300, 256), gen(2)).to(dev), normal((512, 256), gen(3)).to(dev)
    y = torch.full((300, 512), 777.0, dtype=torch.bfloat16, device=dev)
    cache.write(x, x, torch.tensor([99], device=dev))
    assert pkg.lib.o1_gemm(pkg.ptr(a), 256, pkg.ptr(w), None, pkg.ptr(y), 512, 300, 512, 256, 0, None, None, 0, 0.0, 0) == 0
    torch.cuda.synchronize()
    assert pkg.lib.o1_device_error() == 70 and pkg.lib.o1_device_error() == 0
    assert (y != 777.0).float().mean() > 0.99


@gpu
@pytest.mark.parametrize("kind", ["bf16", "fp8", "int8"])
@pytest.mark.parametrize("rows", [3, 3000])
def test_nothing_is_written_after_a_failure(pkg, dev, kind, rows):
    """A kernel before this one fails while the write waits for it: its rows may be stale and stay out of the cache."""
    from latefail import late_failure
    cache = pkg.KvCache(1 + rows // 32, 32, kind, 8, dev)
    x = normal((rows, 8, D), gen(1)).to(dev)
    slots = torch.arange(rows, device=dev)
    cache.write(x, x, torch.full_like(slots, -1))
    torch.cuda.synchronize()
    late_failure(pkg, 98)
    cache.write(x, x, slots)
    torch.cuda.synchronize()
    assert pkg.lib.o1_device_error() == 98
    for t in (cache.k, cache.v):
        assert (t.view(torch.uint8) == 0).all()
    if kind != "bf16":
        assert (cache.k_scale == 0).all() and (cache.v_scale == 0).all()
    cache.write(x, x, slots)
    assert (cache.k.view(torch.uint8) != 0).any()


@gpu
@pytest.mark.parametrize("kind", ["bf16", "fp8", "int8"])
@pytest.mark.parametrize("lens,heads", [([40, 700, 3], 4), ([20000], 8), ([1 + i % 20 for i in range(250)], 2)])
def test_no_row_is_appended_after_a_failure(pkg, dev, kind, lens, heads):
    """Whole items, shared ones and an item to a warp; the next call is as ever."""
    from latefail import late_failure
    c = Case(pkg, dev, kind, lens, 2, 32)
    c.fill()
    q = normal((len(lens), 2 * heads, D), gen(3)).to(dev)
    new = normal((len(lens), 2, D), gen(4)).to(dev)
    want, want_l = c.cache.attend(q, c.dtable, c.dlens, lse=True)
    k, v = c.cache.k.view(torch.uint8).clone(), c.cache.v.view(torch.uint8).clone()
    scales = [t.view(torch.int32).clone() for t in (c.cache.k_scale, c.cache.v_scale) if t is not None]
    torch.cuda.synchronize()
    late_failure(pkg, 98)
    c.cache.attend(q, c.dtable, c.dlens, k=new, v=new)
    torch.cuda.synchronize()
    assert pkg.lib.o1_device_error() == 98
    assert torch.equal(c.cache.k.view(torch.uint8), k) and torch.equal(c.cache.v.view(torch.uint8), v)
    assert all(torch.equal(s, t.view(torch.int32)) for s, t in zip(scales, (c.cache.k_scale, c.cache.v_scale)))
    again, again_l = c.cache.attend(q, c.dtable, c.dlens, lse=True)
    assert torch.equal(again, want) and torch.equal(again_l, want_l)


@gpu
@pytest.mark.parametrize("kind", ["bf16", "fp8", "int8"])
@pytest.mark.parametrize("big", [14, 17, 20, 24])
def test_queries_with_one_large_channel(pkg, dev, kind, big):
    """A query's channel of 2^14 to 2^24 where the keys have zeros: the scores are of the others, and as exact as without it."""
    lens = [100, 700]
    c = Case(pkg, dev, kind, lens, 2, 32, std=1.0)
    for x in c.k:
        x[:, :, 0] = 0.0
    c.fill()
    q = normal((2, 8, D), gen(3), 2.0)
    q[:, :, 0] = 2.0 ** big
    out, lse = c.cache.attend(q.to(dev), c.dtable, c.dlens, lse=True)
    c.check(q, out, lse, what=kind)


@gpu
@pytest.mark.parametrize("kind", ["bf16", "fp8", "int8"])
@pytest.mark.parametrize("lens", [[600, 17, 90, 2500, 33, 1, 300, 600], [600] * 32])
def test_a_sequence_alone_and_among_others(pkg, dev, kind, lens):
    """How rows are shared out follows from all lengths, so the bits may differ; alone and among others a sequence's result keeps its bound from 64 bits."""
    c = Case(pkg, dev, kind, lens, 8, 32, seed=3)
    c.fill()
    q = normal((len(lens), 32, D), gen(3), 1.5)
    out, lse = c.cache.attend(q.to(dev), c.dtable, c.dlens, lse=True)
    c.check(q, out, lse, what="together")
    every = c.lens, c.k, c.v
    for b in range(min(len(lens), 8)):
        out, lse = c.cache.attend(q[b:b + 1].to(dev), c.dtable[b:b + 1], c.dlens[b:b + 1], lse=True)
        c.lens, c.k, c.v = every[0][b:b + 1], every[1][b:b + 1], every[2][b:b + 1]
        c.check(q[b:b + 1], out, lse, what=f"sequence {b} alone")


@gpu
def test_caches_of_one_stream_share_a_workspace(pkg, dev):
    """Calls on a stream follow one another: a model's caches, one of each layer, need one workspace."""
    q, pages, lens = normal((2, 16, D), gen(1)).to(dev), torch.zeros(2, 1, dtype=torch.int32, device=dev), torch.ones(2, dtype=torch.int32, device=dev)
    caches = [pkg.KvCache(2, 16, "int8", 1, dev) for _ in range(9)]
    caches[0].attend(q, pages, lens)
    torch.cuda.synchronize()
    at = torch.cuda.memory_allocated()
    for c in caches[1:]:
        c.attend(q, pages, lens)
    torch.cuda.synchronize()
    assert torch.cuda.memory_allocated() - at < 2 ** 20


@gpu
def test_workspaces_of_captures_go_with_their_graphs(pkg, dev):
    """A process that captures again and again does not grow; a graph that lives keeps its own."""
    import gc
    c = Case(pkg, dev, "int8", [5000, 2000], 1, 32)
    c.fill()
    q = normal((2, 8, D), gen(3)).to(dev)
    out = torch.empty_like(q)
    s = torch.cuda.Stream()

    def once():
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=s):
            pkg.use_torch_stream()
            c.cache.attend(q, c.dtable, c.dlens, out=out)
        g.replay()
        torch.cuda.synchronize()
        return g
    try:
        sizes, kept = [], once()
        for _ in range(12):
            once()
            gc.collect()
            sizes.append(torch.cuda.memory_allocated())
        want = c.cache.attend(q, c.dtable, c.dlens)
        kept.replay()
        torch.cuda.synchronize()
    finally:
        pkg.use_torch_stream()
    # (a destroyed graph is reported by a thread of the runtime's, so one or two may be there)
    assert sizes[-1] - sizes[3] < 3 * pkg.lib.o1_kv_attention_workspace_bytes(8, 1), sizes
    assert torch.equal(out, want)


@gpu
def test_a_table_wider_than_an_int_is_refused(pkg, dev):
    """Its width was cut to 32 bits (17 GB, not touched)."""
    c = pkg.KvCache(4, 16, "int8", 2, dev)
    q, lens = normal((1, 4, D), gen(0)).to(dev), torch.ones(1, dtype=torch.int32, device=dev)
    with pytest.raises(pkg.O1Error, match="pages"):
        c.attend(q, torch.empty(1, 2 ** 32 + 1, dtype=torch.int32, device=dev), lens)
    assert pkg.lib.o1_device_error() == 0


@gpu
@pytest.mark.parametrize("kind", ["bf16", "fp8", "int8"])
@pytest.mark.parametrize("rows,heads,page,off,pad", [(19201, 1, 16, 0, 0), (6403, 3, 48, 0, 8), (2405, 8, 64, 0, 0), (2401, 8, 16, 1, 3), (1205, 16, 32, 8, 8), (19999, 1, 128, 3, 1)])
def test_many_rows_written_and_read_back(pkg, dev, kind, rows, heads, page, off, pad):
    """Eight heads of rows to a warp: a last warp that is not full, heads that do not divide eight, rows inside wider ones at any address, rows left out, rows of zeros,
    with a NaN and of 2^120."""
    g = torch.Generator(device=dev).manual_seed(rows)
    pages = -(-rows // page) + 3
    cache = pkg.KvCache(pages, page, kind, heads, dev)
    pitch = 2 * heads * D + pad
    wide = torch.empty(rows * pitch + off, dtype=torch.bfloat16, device=dev).normal_(0, 1, generator=g)
    w = wide[off:].view(rows, pitch)
    k, v = (w[:, i * heads * D:(i + 1) * heads * D].unflatten(1, (heads, D)) for i in (0, 1))
    k[5], v[7], v[9] = 0.0, 2.0 ** 120, -0.0
    k[11, heads - 1, 5], v[rows - 1, 0, 127] = math.nan, math.inf
    slots = torch.randperm(pages * page, generator=g, device=dev)[:rows]
    left_out = torch.zeros(rows, dtype=torch.bool, device=dev)
    left_out[[3, 100, rows - 2]] = True
    asked = torch.where(left_out, -1, slots)
    cache.write(k, v, asked)
    page_at, at = slots // page, slots % page
    want = []
    for x, store, scales in ((k, cache.k, cache.k_scale), (v, cache.v, cache.v_scale)):
        codes, scale = (None if t is None else t.to(dev) for t in quantised(x.cpu(), kind))
        held = store.view(torch.uint8 if kind != "bf16" else torch.int16)[page_at, :, at]
        assert torch.equal(held[~left_out], codes.view(held.dtype)[~left_out])
        assert (held[left_out] == 0).all()
        if kind != "bf16":
            s = scales[page_at, :, at]
            assert torch.equal(torch.isnan(s)[~left_out], torch.isnan(scale)[~left_out]) and torch.equal(s.nan_to_num(0)[~left_out], scale.nan_to_num(0)[~left_out])
            assert (s[left_out] == 0).all()
        want.append(torch.where(left_out[:, None, None], 0.0, value(codes, scale).to(torch.bfloat16) if kind != "bf16" else x.clone()))
    wide.fill_(7.0)
    cache.read(asked, out=(k, v))
    for name, y, x in (("k", k, want[0]), ("v", v, want[1])):
        assert torch.equal(torch.isnan(y), torch.isnan(x)) and torch.equal(y.nan_to_num(7), x.nan_to_num(7)), name
    assert (w[:, 2 * heads * D:] == 7.0).all() and (wide[:off] == 7.0).all()
    assert pkg.lib.o1_device_error() == 0


@gpu
@pytest.mark.parametrize("kind", ["fp8", "int8"])
@pytest.mark.parametrize("lens,kv_heads,group", [([0, 1, 17, 65, 300], 8, 4), ([4097], 2, 8), ([30011], 1, 8), ([700] * 40, 1, 16), ([33] * 300, 4, 3), ([9001, 1, 0, 12000, 3], 2, 24)])
def test_probabilities_keep_sixteen_bits(pkg, dev, kind, lens, kv_heads, group):
    """Codes are exact, and a probability times v's scale is multiplied as two parts of bf16: 2^-17 of itself over fp8 and int8 rows too, so the values that those
    stand for have the bound of bf16 rows."""
    c = Case(pkg, dev, kind, lens, kv_heads, 32, seed=len(lens))
    c.fill()
    q = normal((len(lens), kv_heads * group, D), gen(11), 1.5)
    out, lse = c.cache.attend(q.to(dev), c.dtable, c.dlens, lse=True)
    c.k, c.v = ([value(*quantised(x, kind)) for x in rows] for rows in (c.k, c.v))
    c.kind = "bf16"
    c.check(q, out, lse, what=kind)


@gpu
@pytest.mark.parametrize("kind", ["bf16", "fp8", "int8", "uint4"])
def test_memory_of_another_gpu_is_refused(pkg, dev, kind):
    c = pkg.KvCache(4, 16, kind, 2, dev)
    x, s = normal((3, 2, D), gen(0)).to(dev), torch.arange(3, device=dev)
    c.write(x, x, s)
    want = c.read(s)
    table, lens = torch.zeros(3, 1, dtype=torch.int32, device=dev), torch.tensor([1, 2, 3], dtype=torch.int32, device=dev)
    real, c._h = c._h, pkg.kvcache._binding.handle(C.addressof(c.c), 2, dev.index + 1)           # (as if its memory were there)
    for call in (lambda: c.write(x, x, s), lambda: c.read(s), lambda: c.attend(x, table, lens)):
        with pytest.raises(pkg.O1Error, match="another GPU than the current one"):
            call()
    c._h = real
    assert all(torch.equal(a, b) for a, b in zip(c.read(s), want))
    pkg.check_cuda_errbuf("after refusals")


@gpu
def test_memory_of_another_gpu_among_two_is_refused(pkg, dev):
    if torch.cuda.device_count() < 2:
        pytest.skip("one GPU")
    c, x, s = pkg.KvCache(4, 16, "bf16", 2, dev), normal((3, 2, D), gen(0)).to(dev), torch.arange(3, device=dev)
    rows = x.flatten(1)
    try:
        torch.cuda.set_device(1)
        for call in (lambda: c.write(x, x, s), lambda: c.read(s), lambda: pkg.residual_norm(rows, rows, None)):
            with pytest.raises(pkg.O1Error, match="another GPU than the current one"):
                call()
    finally:
        torch.cuda.set_device(dev)


@gpu
@pytest.mark.parametrize("kind", ["bf16", "fp8", "int8"])
@pytest.mark.parametrize("lens,kv_heads,group", [([300], 2, 4), ([300], 1, 16), ([100] * 70, 8, 2)])
def test_scores_up_to_the_limit(pkg, dev, kind, lens, kv_heads, group):
    """Scores of up to 2^29: the largest one's row is the result where it is ahead by more than four times a score's error, 2^-19 of its terms' magnitudes.  (A probability has no place for a rounding of
    its maximum by more than 2^7, which is 2^31 of them.)"""
    c = Case(pkg, dev, kind, lens, kv_heads, 32, seed=11)
    c.fill()
    q = normal((len(lens), kv_heads * group, D), gen(3), 2.0 ** 26)
    k, v = (value(*quantised(x[0], kind)).repeat_interleave(group, 1) for x in (c.k, c.v))
    z = torch.einsum("hd,thd->ht", q[0].double(), k) * D ** -0.5
    size = (torch.einsum("hd,thd->ht", q[0].double().abs(), k.abs()) * D ** -0.5).amax(-1)
    assert 2.0 ** 27 < float(z.abs().max()) < 2.0 ** 29
    out, lse = c.cache.attend(q.to(dev), c.dtable, c.dlens, lse=True)
    c.check(q, out, lse, what=kind)
    top = z.topk(2).values
    sure = top[:, 0] - top[:, 1] > 4 * 2.0 ** -19 * size
    assert sure.sum() > len(sure) // 2
    rows, heads = z.argmax(-1)[sure], torch.arange(len(sure))[sure]
    between(out[0, heads], v[rows, heads], v[rows, heads].abs() * 2.0 ** -12, kind)
