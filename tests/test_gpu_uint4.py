"""Rows kept in four bits and the attention over them, against 64-bit arithmetic on the CPU: KvCache with kind "uint4".

The tests of the other kinds (test_gpu_kvcache) run over these rows too, with this file's definition of what is kept and its bounds.  Bounds, from the arithmetic and
not from a run, are as there (a score's error 2^-19 of the sum of its terms' magnitudes, a probability times v's scale 2^-17 of itself, the result rounded
once), but a value is least + code * scale and both products are summed apart, so a value counts with |least| + code * scale in the place of its own magnitude."""
import ctypes as C
import math

import pytest
import torch

import test_gpu_kvcache as base
from test_gpu_kvcache import D, between, gen, normal

gpu = pytest.mark.gpu


def kept(x):
    """Packed codes and (scale, least) of bf16 rows by the definition, in fp32 with its roundings."""
    x = x.float()
    least, most = x.amin(-1) + 0.0, x.amax(-1)
    spread = most - least
    good = torch.isfinite(x).all(-1) & torch.isfinite(spread)
    scale = torch.where(spread >= 2.0 ** -100, spread * torch.tensor(1.0 / 15.0), 0.0).to(torch.bfloat16).float()
    inv = torch.where(good & (scale > 0), torch.ones(()) / scale, 0.0)
    codes = torch.where(good[..., None] & (inv[..., None] > 0), (x - least[..., None]) * inv[..., None], 0.0).round()
    assert codes.min() >= 0 and codes.max() <= 15
    codes = codes.to(torch.uint8)
    pair = torch.stack([torch.where(good, scale, math.nan), torch.where(good, least, math.nan)], -1).to(torch.bfloat16)
    return codes[..., ::2] | codes[..., 1::2] << 4, pair


def unpacked(codes):
    return torch.stack([codes & 15, codes >> 4], -1).flatten(-2)


def quantised(x, kind):
    return kept(x) if kind == "uint4" else OTHERS[0](x, kind)


def value(codes, scale):
    if codes.dtype is not torch.uint8 or scale is None or scale.dtype is not torch.bfloat16:
        return OTHERS[1](codes, scale)
    return scale[..., 1:].double() + unpacked(codes).double() * scale[..., :1].double()


def magnitude(codes, scale):
    return scale[..., 1:].double().abs() + unpacked(codes).double() * scale[..., :1].double()


OTHERS = base.quantised, base.value


class Case4(base.Case):
    def reference(self, q, scale=None):
        B, H = q.shape[:2]
        sc = D ** -0.5 if scale is None else scale
        out, lse = torch.zeros(B, H, D, dtype=torch.float64), torch.full((B, H), -math.inf, dtype=torch.float64)
        tol_o, tol_l = torch.zeros_like(out), torch.zeros_like(lse)
        for b, n in enumerate(self.lens):
            if n == 0:
                continue
            held = [kept(x[b]) for x in (self.k, self.v)]
            (k, v), (ka, va) = ([f(*h).repeat_interleave(H // self.hk, 1) for h in held] for f in (value, magnitude))
            qd = q[b].double()
            z = torch.einsum("hd,thd->ht", qd, k) * sc
            size = (torch.einsum("hd,thd->ht", qd.abs(), ka) * sc).amax(-1)
            lse[b] = torch.logsumexp(z, -1)
            p = torch.exp(z - lse[b][:, None])
            out[b] = torch.einsum("ht,thd->hd", p, v)
            rel = 2.0 * 2.0 ** -19 * size + 2.0 ** -17 + 2.0 ** -18
            tol_o[b] = torch.einsum("ht,thd->hd", p, va) * rel[:, None] + 1e-30
            tol_l[b] = 2.0 ** -19 * size + 2.0 ** -21 * (1 + lse[b].abs())
        return out, lse, tol_o, tol_l


@pytest.fixture(autouse=True)
def four_bits(monkeypatch):
    monkeypatch.setattr(base, "Case", Case4)
    monkeypatch.setattr(base, "quantised", quantised)
    monkeypatch.setattr(base, "value", value)


def test_the_definition():
    """Every value within half a scale (0.53 where code 15 is off by the scale's rounding), the least one exact, ties to even, codes in range."""
    x = normal((500, D), gen(1), 3.0) + torch.randint(-3, 4, (500, 1), generator=gen(2)).bfloat16() * 8
    x[0], x[1, 3:], x[2] = 0.0, 5.0, 1.0e30
    x[3, :16] = torch.arange(16).bfloat16()
    x[3, 16:] = 7.5                                # a tie: to 8
    codes, pair = kept(x)
    got, scale = value(codes, pair), pair[..., 0].double()
    assert ((got - x.double()).abs() <= 0.53125 * scale[:, None]).all()
    assert (got.amin(-1) == x.double().amin(-1)).all()
    assert unpacked(codes)[3].tolist() == list(range(16)) + [8] * 112 and pair[3].tolist() == [1.0, 0.0]
    assert (scale[[0, 2]] == 0).all()


# ------------------------------------------------------------------ rows
def check_rows(pkg, dev, cache, k, v, slots, left_out=None):
    page, pages = cache.page_size, cache.pages
    page_at, at = slots // page, slots % page
    for x, y, store, scales in ((k, 0, cache.k, cache.k_scale), (v, 1, cache.v, cache.v_scale)):
        codes, pair = (t.to(dev) for t in kept(x.cpu()))
        held, s = store[page_at, :, at], scales[page_at, :, at]
        if left_out is not None:
            codes[left_out], pair[left_out] = 0, 0.0
        assert torch.equal(held, codes)
        assert torch.equal(torch.isnan(s), torch.isnan(pair)) and torch.equal(s.nan_to_num(0), pair.nan_to_num(0))
        want = (pair[..., 1:].float() + unpacked(codes).float() * pair[..., :1].float()).to(torch.bfloat16)
        got = cache.read(slots if left_out is None else torch.where(left_out, -1, slots))[y]
        assert torch.equal(torch.isnan(got), torch.isnan(want)) and torch.equal(got.nan_to_num(7), want.nan_to_num(7))
    rest = torch.ones(pages * page, dtype=torch.bool, device=dev)
    rest[slots] = False
    for t in (cache.k, cache.v):
        assert (t.permute(0, 2, 1, 3).reshape(pages * page, -1)[rest] == 0).all()
    for t in (cache.k_scale, cache.v_scale):
        assert (t.permute(0, 2, 1, 3).reshape(pages * page, -1)[rest] == 0).all()


@gpu
@pytest.mark.parametrize("rows,heads,page", [(1, 1, 16), (1, 8, 64), (37, 8, 48), (515, 3, 16), (64, 16, 128), (19201, 1, 16), (2405, 8, 64), (6403, 3, 48)])
def test_rows_written_and_read_back(pkg, dev, rows, heads, page):
    g = gen(rows + heads)
    pages = -(-rows // page) + 3
    cache = pkg.KvCache(pages, page, "uint4", heads, dev)
    k, v = normal((rows, heads, D), g, 2.0), normal((rows, heads, D), g) + 100.0
    k[:, :, ::13] *= 50
    if rows > 6:
        k[0], v[1], k[2, 0], v[2], k[4], v[4] = 0.0, 2.0 ** -130, -0.0, -3.0, k[4] * 2.0 ** -101, v[4] * 2.0 ** -106
        v[3] = 2.0 ** 120
        k[3] = torch.linspace(-1.6e38, 1.6e38, D).bfloat16()
        k[5, 0, 0], k[5, 0, 1] = 3.0e38, -3.0e38                 # a spread beyond fp32
        k[1, 0, 5], v[2, heads - 1, 7], v[3, 0, 0], v[5, 0] = math.nan, math.inf, -math.inf, -math.inf
    slots = torch.randperm(pages * page, generator=g)[:rows].to(dev)
    cache.write(k.to(dev), v.to(dev), slots)
    check_rows(pkg, dev, cache, k, v, slots)
    assert pkg.lib.o1_device_error() == 0


@gpu
@pytest.mark.parametrize("rows,heads,page,off,pad", [(2401, 8, 16, 1, 3), (1205, 16, 32, 8, 8), (19999, 1, 128, 3, 1), (30, 2, 16, 5, 7)])
def test_rows_inside_wider_ones_and_rows_left_out(pkg, dev, rows, heads, page, off, pad):
    g = torch.Generator(device=dev).manual_seed(rows)
    pages = -(-rows // page) + 3
    cache = pkg.KvCache(pages, page, "uint4", heads, dev)
    pitch = 2 * heads * D + pad
    wide = torch.empty(rows * pitch + off, dtype=torch.bfloat16, device=dev).normal_(0, 1, generator=g)
    w = wide[off:].view(rows, pitch)
    k, v = (w[:, i * heads * D:(i + 1) * heads * D].unflatten(1, (heads, D)) for i in (0, 1))
    slots = torch.randperm(pages * page, generator=g, device=dev)[:rows]
    left_out = torch.zeros(rows, dtype=torch.bool, device=dev)
    left_out[[3, 10, rows - 2]] = True
    cache.write(k, v, torch.where(left_out, -1, slots))
    check_rows(pkg, dev, cache, k, v, slots, left_out)
    want = cache.read(slots)
    wide.fill_(7.0)
    cache.read(slots, out=(k, v))
    assert torch.equal(k, want[0]) and torch.equal(v, want[1])
    assert (w[:, 2 * heads * D:] == 7.0).all() and (wide[:off] == 7.0).all()


@gpu
def test_negative_and_wrong_slots(pkg, dev):
    cache = pkg.KvCache(2, 16, "uint4", 2, dev)
    x = normal((4, 2, D), gen(1)).to(dev)
    cache.write(x, x, torch.tensor([-1, 3, -5, 31], device=dev))
    k, v = cache.read(torch.tensor([3, -2, 31, 0], device=dev))
    assert pkg.lib.o1_device_error() == 0
    assert (k[1] == 0).all() and (v[1] == 0).all() and (k[3] == 0).all() and (k[0] != 0).any()
    before, scales = cache.k.clone(), cache.k_scale.clone()
    cache.write(x, x, torch.tensor([32, -1, -1, 2 ** 40], device=dev))
    assert pkg.lib.o1_device_error() == 70
    assert torch.equal(before, cache.k) and torch.equal(scales, cache.k_scale)
    k, _ = cache.read(torch.tensor([32], device=dev))
    assert (k == 0).all() and pkg.lib.o1_device_error() == 70


# ------------------------------------------------------------------ the other kinds' tests, over these rows
@gpu
@pytest.mark.parametrize("kv_heads,group,page", [(8, 4, 16), (1, 1, 16), (2, 8, 64), (3, 3, 48), (2, 7, 32), (1, 16, 128), (2, 12, 16), (1, 24, 64), (1, 33, 16), (16, 1, 32),
                                                 (8, 4, 64), (4, 2, 96)])
def test_attention_of_ragged_sequences(pkg, dev, kv_heads, group, page):
    base.test_attention_of_ragged_sequences(pkg, dev, "uint4", kv_heads, group, page)


@gpu
@pytest.mark.parametrize("lens,kv_heads,group", [([1], 1, 1), ([1], 8, 4), ([85], 8, 4), ([4097], 8, 4), ([30011], 1, 8), ([30011], 2, 16), ([9001, 1, 0, 12000, 3], 2, 4),
                                                 ([700] * 40, 1, 4), ([0, 0, 0], 2, 2), ([257] * 300, 1, 2), ([1] * 700 + [5000], 1, 1)])
def test_attention_over_few_and_many_rows(pkg, dev, lens, kv_heads, group):
    base.test_attention_over_few_and_many_rows(pkg, dev, "uint4", lens, kv_heads, group)


@gpu
@pytest.mark.parametrize("lens,kv_heads,group,page", [([1, 16, 17, 0, 33, 128, 2, 129], 8, 4, 16), ([1], 8, 4, 64), ([20000], 2, 4, 64), ([5, 700, 1300], 1, 24, 48),
                                                      ([3] * 90, 4, 1, 16), ([64, 65, 63, 127, 128, 49], 2, 4, 32), ([64, 65, 63, 127, 128, 49], 2, 16, 128)])
def test_new_rows_appended_by_the_same_call(pkg, dev, lens, kv_heads, group, page):
    base.test_new_rows_appended_by_the_same_call(pkg, dev, "uint4", lens, kv_heads, group, page)


@gpu
@pytest.mark.parametrize("batch,kv_heads,group,page,most", base.MANY)
def test_many_short_sequences(pkg, dev, batch, kv_heads, group, page, most):
    base.test_many_short_sequences(pkg, dev, "uint4", batch, kv_heads, group, page, most)


@gpu
@pytest.mark.parametrize("batch,kv_heads,group,page,most", [(300, 4, 4, 16, 90), (230, 2, 16, 32, 33), (470, 1, 1, 48, 48)])
def test_many_short_sequences_with_new_rows(pkg, dev, batch, kv_heads, group, page, most):
    base.test_many_short_sequences_with_new_rows(pkg, dev, "uint4", batch, kv_heads, group, page, most)


@gpu
def test_scores_of_any_size(pkg, dev):
    base.test_scores_of_any_size(pkg, dev, "uint4")


@gpu
def test_not_finite_rows_stay_where_they_are(pkg, dev):
    base.test_not_finite_rows_stay_where_they_are(pkg, dev, "uint4")


@gpu
@pytest.mark.parametrize("rows", [3, 3000])
def test_nothing_is_written_after_a_failure(pkg, dev, rows):
    base.test_nothing_is_written_after_a_failure(pkg, dev, "uint4", rows)


@gpu
@pytest.mark.parametrize("lens,heads", [([40, 700, 3], 4), ([20000], 8), ([1 + i % 20 for i in range(250)], 2)])
def test_no_row_is_appended_after_a_failure(pkg, dev, lens, heads):
    base.test_no_row_is_appended_after_a_failure(pkg, dev, "uint4", lens, heads)


@gpu
@pytest.mark.parametrize("big", [14, 24])
def test_queries_with_one_large_channel(pkg, dev, big):
    base.test_queries_with_one_large_channel(pkg, dev, "uint4", big)


@gpu
@pytest.mark.parametrize("lens", [[600, 17, 90, 2500, 33, 1, 300, 600], [600] * 32])
def test_a_sequence_alone_and_among_others(pkg, dev, lens):
    base.test_a_sequence_alone_and_among_others(pkg, dev, "uint4", lens)


# ------------------------------------------------------------------ what four bits add
# More items than half of the teams, and much work: parts to warps, an item joined from as many as have some of it (of the longest one from more than a thousand, in groups).
AMONG = [([1] * 120 + [100000] + [3] * 120, 1, 2, 32), ([2] * 130 + [20000, 0, 9000] + [70] * 110, 1, 8, 64), ([64 + 61 * (i % 40) for i in range(120)], 2, 4, 48),
         ([500 + i for i in range(150)], 2, 12, 16)]


@gpu
@pytest.mark.parametrize("lens,kv_heads,group,page", AMONG)
def test_long_sequences_among_many(pkg, dev, lens, kv_heads, group, page):
    c = Case4(pkg, dev, "uint4", lens, kv_heads, page, seed=len(lens))
    c.fill()
    q = normal((len(lens), kv_heads * group, D), gen(13), 1.5)
    out, lse = c.cache.attend(q.to(dev), c.dtable, c.dlens, lse=True)
    c.check(q, out, lse)
    for _ in range(3):
        again, lse2 = c.cache.attend(q.to(dev), c.dtable, c.dlens, lse=True)
        assert torch.equal(out, again) and torch.equal(lse, lse2)
    assert torch.equal(out, c.cache.attend(q.to(dev), c.dtable, c.dlens))


@gpu
@pytest.mark.parametrize("rows,batch,group", [(100000, 450, 1), (30000, 450, 4), (30000, 300, 7), (100000, 1, 4)])
def test_long_sums_keep_their_bits(pkg, dev, rows, batch, group):
    """Hundreds of chunks a warp with scores that hardly differ: codes are not negative, so that their sums grow all the way, and the tensor cores cut what they add; the error stays
    that of a short sequence.  (All sequences have the same rows.)"""
    c = Case4(pkg, dev, "uint4", [rows], 1, 64, seed=9, width_extra=0)
    c.fill()
    q = normal((batch, group, D), gen(3), 0.05)
    out, lse = c.cache.attend(q.to(dev), c.dtable.expand(batch, -1).contiguous(), c.dlens.expand(batch).contiguous(), lse=True)
    held = [kept(x[0][:, 0]) for x in (c.k, c.v)]
    (k, v), (ka, va) = ([f(*h) for h in held] for f in (value, magnitude))
    some = slice(0, 450, 29)
    qd = q[some].double()
    z = qd @ k.T * D ** -0.5
    ref = torch.logsumexp(z, -1)
    p = torch.exp(z - ref[..., None])
    size = (qd.abs() @ ka.T * D ** -0.5).amax(-1)
    between(out[some], p @ v, (p @ va) * (2.0 * 2.0 ** -19 * size + 2.0 ** -17 + 2.0 ** -18)[..., None], "out")
    assert ((lse[some].cpu().double() - ref).abs() <= 2.0 ** -19 * size + 2.0 ** -21 * (1 + ref.abs())).all()


@gpu
def test_long_sums_lean_to_no_side(pkg, dev):
    """400 chunks a warp.  What is left of the error is the result's rounding: at most half a step, 2^-8 of the value, to either side alike, so that its square is (2^-8 x)^2 / 3 at most on
    average and the mean over the 128 columns (the sequences' results are close to one another and count as one) within 6 deviations of 0.  Cut sums lean to one side by three times that."""
    c = Case4(pkg, dev, "uint4", [100000], 1, 64, seed=9, width_extra=0)
    c.fill()
    q = normal((450, 1, D), gen(3), 0.05)
    out = c.cache.attend(q.to(dev), c.dtable.expand(450, -1).contiguous(), c.dlens.expand(450).contiguous())
    k, v = (value(*kept(x[0][:, 0])) for x in (c.k, c.v))
    qd = q[:20].double()
    ref = torch.softmax(qd @ k.T * D ** -0.5, -1) @ v
    error = out[:20].cpu().double() - ref
    assert abs(error.mean().item()) <= 6 * 2.0 ** -8 * (ref.square().mean().item() / 3 / D) ** 0.5


@gpu
@pytest.mark.parametrize("lens,kv_heads,group,page", [AMONG[0], AMONG[2]])
def test_new_rows_of_long_sequences_among_many(pkg, dev, lens, kv_heads, group, page):
    base.test_new_rows_appended_by_the_same_call(pkg, dev, "uint4", [n for n in lens], kv_heads, group, page)


@gpu
def test_many_sequences_with_wrong_tables(pkg, dev):
    for lens, page in (([1 + b % 40 for b in range(260)], 16), ([300 + b for b in range(150)], 32)):
        c = Case4(pkg, dev, "uint4", lens, 2, page)
        c.fill()
        n = len(lens)
        q = normal((n, 8, D), gen(1)).to(dev)
        good = c.cache.attend(q, c.dtable, c.dlens)
        assert pkg.lib.o1_device_error() == 0
        t, ln = c.dtable.clone(), c.dlens.clone()
        t[100, 0], t[7, 0] = c.cache.pages, -1
        out = c.cache.attend(q, t, c.dlens)
        rest = [b for b in range(n) if b not in (7, 100)]
        assert pkg.lib.o1_device_error() == 70 and torch.equal(out[rest], good[rest])
        ln[100], ln[7] = -1, page * c.table.shape[1] + 1
        out = c.cache.attend(q, c.dtable, ln)
        # (lengths decide how rows are shared out: the others within their bounds, not the same bits)
        assert pkg.lib.o1_device_error() == 71 and (out[[7, 100]] == 0).all()
        c.lens = [0 if b in (7, 100) else x for b, x in enumerate(lens)]
        c.k, c.v = ([x[:k] for x, k in zip(rows, c.lens)] for rows in (c.k, c.v))
        c.check(q.cpu(), out)


@gpu
@pytest.mark.parametrize("group", [1, 4, 5, 8, 16])
def test_values_of_very_different_sizes(pkg, dev, group):
    """Values of 2^-90 to 2^90 from row to row: rows that count for nothing take no bits from those that count, whichever come first."""
    lens = [700, 700, 65, 900]
    c = Case4(pkg, dev, "uint4", lens, 2, 32, seed=5, std=6.0)
    for b, n in enumerate(lens):
        size = torch.linspace(-90, 90, n).flip(0) if b % 2 else torch.linspace(-90, 90, n)
        c.v[b] = (c.v[b].double() * torch.exp2(size[:, None, None].double())).to(torch.bfloat16)
    c.v[3][::2] = 0.0
    c.fill()
    q = normal((4, 2 * group, D), gen(3), 4.0)
    out, lse = c.cache.attend(q.to(dev), c.dtable, c.dlens, lse=True)
    c.check(q, out, lse)


@gpu
@pytest.mark.parametrize("group", [2, 8, 12])
def test_rows_far_from_zero_and_constant_rows(pkg, dev, group):
    """Values to one side of zero, rows of one value (no codes), rows of zeros."""
    lens = [130, 1, 64, 300]
    c = Case4(pkg, dev, "uint4", lens, 1, 16, seed=6)
    c.v[0], c.k[0] = c.v[0] + 50.0, c.k[0] - 3.0
    c.v[1][:], c.k[1][:] = -2.5, 0.75
    c.v[2][:] = 0.0
    c.v[3][::3], c.k[3][1::3] = 9.0, 0.0
    c.fill()
    q = normal((4, group, D), gen(3), 0.5)
    out, lse = c.cache.attend(q.to(dev), c.dtable, c.dlens, lse=True)
    c.check(q, out, lse)


@gpu
@pytest.mark.parametrize("lens,kv_heads,group", [([70, 700], 1, 4), ([300, 5], 2, 8), ([900, 64], 1, 16), ([100] * 300, 2, 4)])
def test_queries_that_are_not_finite_or_huge(pkg, dev, lens, kv_heads, group):
    """A NaN or Inf in a query's head reaches that head's result and no other; queries of 2^-120 and 2^120 among others."""
    c = Case4(pkg, dev, "uint4", lens, kv_heads, 32, seed=8)
    c.fill()
    q = normal((len(lens), kv_heads * group, D), gen(3), 1.5)
    want, want_l = c.cache.attend(q.to(dev), c.dtable, c.dlens, lse=True)
    bad = q.clone()
    bad[0, 1, 5], bad[1, 0, 127], bad[1, 3] = math.nan, math.inf, q[1, 3] * 2.0 ** -120
    out, lse = c.cache.attend(bad.to(dev), c.dtable, c.dlens, lse=True)
    for b, h in ((0, 1), (1, 0)):
        assert not torch.isfinite(out[b, h].float()).any() and not torch.isfinite(lse[b, h])
    keep = torch.ones(q.shape[:2], dtype=torch.bool)
    keep[0, 1] = keep[1, 0] = keep[1, 3] = False
    assert torch.equal(out[keep.to(dev)], want[keep.to(dev)]) and torch.equal(lse[keep.to(dev)], want_l[keep.to(dev)])
    bad = q.clone()
    bad[1, 3], bad[0, 2] = q[1, 3] * 2.0 ** -120, 0.0
    bad[0, 0] = q[0, 0] * 2.0 ** 120          # its largest score takes all
    out, lse = c.cache.attend(bad.to(dev), c.dtable, c.dlens, lse=True)
    assert torch.isfinite(out.float()).all()
    got, ref = out[0, 0].cpu().double(), value(*kept(c.v[0][:, 0]))
    assert ((got[None] - ref).abs().amax(1) <= 2.0 ** -8 * ref.abs().amax()).any()
    q[0, 0] = 0.0
    bad[0, 0] = 0.0
    out, lse = c.cache.attend(bad.to(dev), c.dtable, c.dlens, lse=True)
    c.check(bad, out, lse)


@gpu
def test_offsets_past_32_bits(pkg, dev):
    """A cache of more than 2^32 bytes of codes, with rows at its end."""
    heads, page = 8, 128
    pages = 2 ** 33 // (heads * page * D) + 40
    cache = pkg.KvCache(pages, page, "uint4", heads, dev)
    c = Case4(pkg, dev, "uint4", [300, 128], heads, page, width_extra=0)
    c.cache = cache
    c.table += pages - 10
    c.table[c.table >= pages] = 0
    c.dtable = c.table.to(dev)
    c.fill()
    k, _ = cache.read(c.slots(0).to(dev))
    assert torch.equal(k.cpu().double(), value(*kept(c.k[0])).to(torch.bfloat16).double())
    q = normal((2, 32, D), gen(3))
    c.check(q, c.cache.attend(q.to(dev), c.dtable, c.dlens))


@gpu
def test_streams_graphs_and_wrong_tables(pkg, dev):
    lens = [3000, 17, 900]
    c = Case4(pkg, dev, "uint4", lens, 4, 32)
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
        ln, out = c.dlens.clone(), torch.empty_like(want)
        with torch.cuda.stream(streams[0]):
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph, stream=streams[0]):
                pkg.use_torch_stream()
                c.cache.attend(q, c.dtable, ln, out=out)
        ln.copy_(torch.tensor([100, 0, 33], dtype=torch.int32))
        graph.replay()
        torch.cuda.synchronize()
    finally:
        pkg.use_torch_stream()
    assert torch.equal(out, c.cache.attend(q, c.dtable, ln))
    for page in (c.cache.pages, -1, 2 ** 31 - 1, -2 ** 31):
        t = c.dtable.clone()
        t[0, 1] = page
        got = c.cache.attend(q, t, c.dlens)
        assert pkg.lib.o1_device_error() == 70 and torch.equal(got[1:], want[1:])
    new, before = normal((3, 4, D), gen(2)).to(dev), c.cache.k.clone()
    for n in (-1, 32 * c.table.shape[1] + 1, 2 ** 31 - 1, -2 ** 31):
        bad = c.dlens.clone()
        bad[0] = n
        got = c.cache.attend(q, c.dtable, bad)
        assert pkg.lib.o1_device_error() == 71 and torch.equal(got[1:], want[1:]) and (got[0] == 0).all()
    bad = torch.tensor([-3, 2 ** 30, 0], dtype=torch.int32, device=dev)
    c.cache.attend(q, c.dtable, bad, k=new, v=new)
    assert pkg.lib.o1_device_error() == 71 and torch.equal(before, c.cache.k)


@gpu
def test_arguments_that_do_not_fit(pkg, dev):
    E = pkg.O1Error
    c = pkg.KvCache(4, 16, "uint4", 2, dev)
    assert c.k.shape == (4, 2, 16, 64) and c.k_scale.shape == (4, 2, 16, 2) and c.k_scale.dtype is torch.bfloat16
    same = pkg.KvCache.over(c.k, c.v, c.k_scale, c.v_scale)
    assert same.c.type == 4
    for args in ((c.k, c.v), (c.k, c.v, c.k_scale[..., 0], c.v_scale), (c.k, c.v, c.k_scale.float(), c.v_scale)):
        with pytest.raises(E, match="scales"):
            pkg.KvCache.over(*args)
    with pytest.raises(E, match="wanted"):
        pkg.KvCache.over(c.k[..., :32].contiguous(), c.v[..., :32].contiguous(), c.k_scale, c.v_scale)
    wide = torch.zeros(4, 2, 16, 128, dtype=torch.uint8, device=dev)
    with pytest.raises(E, match="wanted"):
        pkg.KvCache.over(wide, wide, c.k_scale, c.v_scale)
    with pytest.raises(E, match="multiple of 16"):
        pkg.KvCache(4, 24, "uint4", 2, dev)
    x, s = normal((3, 2, D), gen(0)).to(dev), torch.arange(3, device=dev)
    for bad in (x.float(), x[:, :1], x[..., :64], x.cpu()):
        with pytest.raises(E, match="KvCache.write"):
            c.write(bad, x, s)


def test_entry_points_refuse_before_they_touch_the_gpu(pkg):
    K, one = pkg.KvCacheC, C.c_void_p(4096)
    good = dict(k=4096, v=4096, k_scale=4096, v_scale=4096, type=4, pages=4, page_size=16, kv_heads=2, head_dim=128)
    for want, change in ((6, dict(k=None)), (6, dict(k_scale=None)), (6, dict(v_scale=None)), (9, dict(head_dim=64)), (9, dict(page_size=8)), (9, dict(v_scale=4100)), (9, dict(type=5))):
        assert pkg.lib.o1_kv_write(C.byref(K(**{**good, **change})), one, 256, one, 256, one, 1) == want, change
        assert b"kv_write" in pkg.lib.hd_cuda_last_error()
    pkg.lib.hd_cuda_clear_error()


# ------------------------------------------------------------------ bits of the sums
@gpu
@pytest.mark.parametrize("kv_heads,group,batch", [(1, 1, 40), (2, 4, 40), (1, 8, 40), (8, 1, 60), (8, 4, 60), (8, 8, 60)])
def test_values_in_the_middle_of_their_rows(pkg, dev, kv_heads, group, batch):
    """Rows of -7.5, 7.5 and half ones (a scale of 1, codes 7 and 8), each key twice with the halves' signs turned: exactly zero in all but two columns.  What a probability loses to 16 bits takes
    the codes' middle with it, so that only sums in fp32 are left: 2^-19 of the codes' (as for scores) and 2^-20 of the least values' (16 additions), 7.5 each.  (62 of 64 rows weigh the same, and
    16 bits of a weight are off by up to 2^-17: 5.7e-5 where the bound is 2.1e-5.)"""
    c = Case4(pkg, dev, "uint4", [64] * batch, kv_heads, 64, seed=3, width_extra=0)
    sign = torch.where((torch.arange(64)[:, None] + torch.arange(D)) % 2 > 0, 0.5, -0.5).bfloat16()
    sign[:, 0], sign[:, 1] = -7.5, 7.5
    for b in range(batch):
        c.k[b][:2], c.k[b][2:] = c.k[b][:1], c.k[b][2:3]
        c.v[b][:] = sign[:, None]
    c.fill()
    q = normal((batch, kv_heads * group, D), gen(3), 0.4)
    out, lse = c.cache.attend(q.to(dev), c.dtable, c.dlens, lse=True)
    c.check(q, out, lse)
    assert float(out[..., 2:].float().abs().max()) <= 7.5 * (2.0 ** -19 + 2.0 ** -20)


# ------------------------------------------------------------------ the range of queries
def one_row_takes_all(c, q, out, lse, scale):
    """A score's error is 2^-19 of the sum of its terms' magnitudes: where the largest one is ahead by four times that, its row is the result and its score the log-sum-exp."""
    ref, ref_l, _, tol_l = c.reference(q, scale)
    n = c.lens[0]
    (k, ka), (v, va) = ([f(*kept(x[0])).repeat_interleave(q.size(1) // c.hk, 1) for f in (value, magnitude)] for x in (c.k, c.v))
    z = torch.einsum("hd,thd->ht", q[0].double(), k)
    size = torch.einsum("hd,thd->ht", q[0].double().abs(), ka).amax(-1)
    top = z.topk(2).values
    sure = top[:, 0] - top[:, 1] > 4 * 2.0 ** -19 * size
    assert sure.sum() > len(sure) // 2 and n > 1
    heads, rows = torch.arange(len(sure))[sure], z.argmax(-1)[sure]
    between(out[0, heads], v[rows, heads], 2.0 ** -17 * va[rows, heads], "out")
    assert ((lse.cpu().double() - ref_l).abs() <= tol_l)[0].all()


@gpu
@pytest.mark.parametrize("scale,top", [(None, 121), (None, 123), (None, 124), (1.0, 120), (1.0, 121), (2.0 ** 40, 81), (2.0 ** 70, 51), (2.0 ** 114, 7), (2.0 ** -60, 120), (2.0 ** -100, 100)])
@pytest.mark.parametrize("lens,kv_heads,group", [([300], 2, 4), ([300], 1, 8), ([300] * 60, 8, 2)])
def test_queries_up_to_the_limit(pkg, dev, lens, kv_heads, group, scale, top):
    """scale times the largest query up to 2^121: one row takes all (with the smaller scales some do), and nothing on the way leaves fp32."""
    c = Case4(pkg, dev, "uint4", lens, kv_heads, 32, seed=11)
    if scale is not None and scale > 2.0 ** 100:
        c.k = [(x.float() * 2.0 ** -20).to(torch.bfloat16) for x in c.k]         # (scores of fp32's range)
    c.fill()
    q = normal((len(lens), kv_heads * group, D), gen(3))
    q = (q.float() / q.float().abs().amax(-1, keepdim=True) * 2.0 ** top).to(torch.bfloat16)
    assert float(q.float().abs().max()) == 2.0 ** top
    out, lse = c.cache.attend(q.to(dev), c.dtable, c.dlens, lse=True, scale=scale)
    c.check(q, out, lse, scale=scale)
    if (scale or D ** -0.5) * 2.0 ** top > 2.0 ** 30:
        one_row_takes_all(c, q, out, lse, scale)


def test_scales_beyond_the_limit_are_refused(pkg):
    one = C.c_void_p(4096)
    good = dict(k=4096, v=4096, k_scale=4096, v_scale=4096, type=4, pages=4, page_size=16, kv_heads=2, head_dim=128)
    for scale in (2.0 ** 114.5, 3.0e38, math.inf, math.nan, 0.0, -1.0):
        k = pkg.KvCacheC(**good)
        assert pkg.lib.o1_kv_attention(C.byref(k), one, 256, None, 0, None, 0, one, 4, 4, one, one, 256, None, 1, 2, scale, one, 1 << 30) == 9, scale
        assert b"scale" in pkg.lib.hd_cuda_last_error()
    pkg.lib.hd_cuda_clear_error()


@gpu
@pytest.mark.parametrize("spread", [False, True])
@pytest.mark.parametrize("top,scale", [(124, None), (121, 1.0), (123, 2.0 ** -20), (127, 2.0 ** -6), (127, 2.0 ** -30), (60, None), (-60, None), (-110, None)])
@pytest.mark.parametrize("lens,kv_heads,group", [([300, 41], 2, 4), ([300, 64], 1, 8), ([100] * 60, 8, 2)])
def test_queries_of_one_sign(pkg, dev, lens, kv_heads, group, scale, top, spread):
    """A head's queries of one sign, whose sum is up to 128 times the largest of them, and keys as small (or as large) as they are large, so that scores are ordinary: rows of one value, of which the
    sum alone makes the scores, and with a value of another size in one column."""
    c = Case4(pkg, dev, "uint4", lens, kv_heads, 32, seed=12)
    for b, x in enumerate(c.k):
        one = x.float()[..., :1].expand(x.shape).clone()
        if spread:
            one[..., 5] = one[..., 5] * 3 + 40
        c.k[b] = (one * 2.0 ** -top * 0.05 / (scale or D ** -0.5)).to(torch.bfloat16)
    c.fill()
    q = normal((len(lens), kv_heads * group, D), gen(3)).float().abs().clamp(0.5, 2.0) * 2.0 ** (top - 1)
    q[:, ::2] *= -1
    q = q.to(torch.bfloat16)
    assert torch.isfinite(q.float()).all() and float(q.float().abs().max()) == 2.0 ** top
    out, lse = c.cache.attend(q.to(dev), c.dtable, c.dlens, lse=True, scale=scale)
    c.check(q, out, lse, scale=scale)


@gpu
def test_parts_of_warps_are_joined_when_all_have_come(pkg, dev):
    """One item in more than a thousand warps' parts (two levels of joins) among others of two and more, many times over and launch upon launch: the same bits each time, with nothing left of the
    launch before, whose queries are others."""
    lens = [1] * 120 + [100000] + [700 + 3 * i for i in range(120)]
    c = Case4(pkg, dev, "uint4", lens, 2, 32, seed=14)
    c.fill()
    qs = [normal((len(lens), 8, D), gen(i), 1.5) for i in (1, 2)]
    on_gpu = [q.to(dev) for q in qs]
    first = [c.cache.attend(q, c.dtable, c.dlens, lse=True) for q in on_gpu]
    c.check(qs[0], *first[0])
    again = [[c.cache.attend(q, c.dtable, c.dlens, lse=True) for q in on_gpu] for _ in range(60)]
    for pair in again:
        for got, want in zip(pair, first):
            assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


# ------------------------------------------------------------------ workspaces
def test_workspaces_by_kind(pkg):
    """Two counters of four bytes for the two parts of 1920 warps, then 130 values for each head of the two parts of 480 teams, whatever the kind, or (four bits, at most eight heads) of the warps."""
    lib = pkg.lib
    for heads, kv_heads in ((1, 1), (32, 8), (16, 2), (16, 1), (32, 1), (128, 2)):
        group = heads // kv_heads
        plain = lib.o1_kv_attention_workspace_bytes(heads, kv_heads)
        assert plain == 1920 * 2 * 8 + 480 * 2 * min(group, 16) * 130 * 4
        assert [lib.o1_kv_attention_workspace_bytes_of(t, heads, kv_heads) for t in (0, 1, 2)] == [plain] * 3
        assert lib.o1_kv_attention_workspace_bytes_of(4, heads, kv_heads) == 1920 * 2 * 8 + 1920 * 2 * min(group, 8) * 130 * 4 > plain
    for args in ((3, 4, 2), (5, 4, 2), (-1, 4, 2), (0, 4, 3), (4, 0, 1), (4, 4, 0)):
        assert lib.o1_kv_attention_workspace_bytes_of(*args) == -1
    dims = (9, 32, 8, 4096, 12288, 128)
    plain = lib.o1_decode_scratch_bytes(*dims)
    assert plain == lib.o1_decode_scratch_bytes_of(0, *dims) == lib.o1_decode_scratch_bytes_of(2, *dims) and lib.o1_decode_scratch_bytes_of(3, *dims) == -1
    assert lib.o1_decode_scratch_bytes_of(4, *dims) - plain == lib.o1_kv_attention_workspace_bytes_of(4, 32, 8) - lib.o1_kv_attention_workspace_bytes(32, 8)


def attend_in(pkg, c, q, room):
    """o1_kv_attention in a workspace that the caller has; a guard behind it."""
    at, n = room
    out = torch.empty_like(q)
    pkg.check(pkg.lib.o1_kv_attention(C.byref(c.cache.c), pkg.ptr(q), q.size(1) * D, None, 0, None, 0, pkg.ptr(c.dtable), c.dtable.size(1), c.dtable.size(1), pkg.ptr(c.dlens), pkg.ptr(out),
                                      q.size(1) * D, None, len(c.lens), q.size(1), D ** -0.5, pkg.ptr(at), n), "o1_kv_attention")
    return out


@gpu
@pytest.mark.parametrize("lens,kv_heads,group,page", AMONG + [([60] * 128, 8, 4, 64), ([100000], 2, 4, 64)])
def test_workspaces_of_either_size(pkg, dev, lens, kv_heads, group, page):
    """With the room that any kind needs, and with that of four bits; the larger one also between calls over rows of a byte, which use the same counters.  Nothing behind them is written."""
    c, other = Case4(pkg, dev, "uint4", lens, kv_heads, page, seed=15), Case4(pkg, dev, "int8", [900, 3, 5000], kv_heads, page, seed=16)
    c.fill(), other.fill()
    q, q2 = normal((len(lens), kv_heads * group, D), gen(13), 1.5), normal((3, kv_heads * group, D), gen(14))
    want2 = other.cache.attend(q2.to(dev), other.dtable, other.dlens)
    for size in (pkg.lib.o1_kv_attention_workspace_bytes(kv_heads * group, kv_heads), pkg.lib.o1_kv_attention_workspace_bytes_of(4, kv_heads * group, kv_heads)):
        space = torch.full((size + 4096,), 0xA5, dtype=torch.uint8, device=dev)
        space[:32768] = 0
        outs = []
        for _ in range(2):
            outs.append(attend_in(pkg, c, q.to(dev), (space, size)))
            assert torch.equal(attend_in(pkg, other, q2.to(dev), (space, size)), want2)
        c.check(q, outs[0])
        assert torch.equal(outs[0], outs[1]) and (space[size:] == 0xA5).all() and (space[:30720] == 0).all()
    assert torch.equal(outs[0], c.cache.attend(q.to(dev), c.dtable, c.dlens))
