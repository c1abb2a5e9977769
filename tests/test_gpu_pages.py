"""Pages handed out on the GPU (KvPages, o1_kv_pages_*) against lists on the host; whole numbers, which have to be equal.  At the end pages, rotary positions,
rows of four bits and attention together, as a server uses them."""
import ctypes as C
import math
import random

import pytest
import torch

from test_gpu_kvcache import D, between, normal
from test_gpu_uint4 import kept, magnitude, value

gpu = pytest.mark.gpu


class Model:
    """The same pages on the host, by the definition."""

    def __init__(self, pages, page, seqs, width):
        self.page, self.width, self.size = page, width, pages
        self.free, self.lens, self.table = list(range(pages - 1, -1, -1)), [0] * seqs, [[] for _ in range(seqs)]

    def need(self, n):
        return -(-n // self.page)

    def codes(self, seqs):
        return [70 if not 0 <= s < len(self.lens) or seqs.count(s) > 1 else 0 for s in seqs]

    def grow(self, counts, rows, seqs=None):
        seqs = list(range(len(counts))) if seqs is None else seqs
        starts, lens, tables, slots, positions, bad, left = [0], [], [], [], [], set(), len(self.free)
        for b, (s, n, code) in enumerate(zip(seqs, counts, self.codes(seqs))):
            wanted = 0
            if not code and (n < 0 or self.lens[s] + n > self.width * self.page):
                code = 71
            if not code:
                wanted = self.need(self.lens[s] + n) - self.need(self.lens[s])
            left -= wanted
            end = starts[-1] + max(n, 0)
            if not code and n > 0 and end > rows:
                code = 71
            if not code and wanted and left < 0:
                code = 73
            starts.append(end)
            if code:
                bad.add(code)
                lens.append(0)
                tables.append([])
                slots += [-1] * min(max(n, 0), max(rows - len(slots), 0))
                positions += [0] * (len(slots) - len(positions))
                continue
            self.table[s] += [self.free.pop() for _ in range(wanted)]
            at = range(self.lens[s], self.lens[s] + n)
            slots += [self.table[s][t // self.page] * self.page + t % self.page for t in at]
            positions += at
            self.lens[s] += n
            lens.append(self.lens[s])
            tables.append(list(self.table[s]))
        pad = [-1] * (rows - len(slots)), [0] * (rows - len(slots))
        return (slots + pad[0])[:rows], (positions + pad[1])[:rows], starts, lens, [t + [-1] * (self.width - len(t)) for t in tables], bad

    def shrink(self, keep, seqs=None):
        seqs = list(range(len(keep))) if seqs is None else seqs
        bad, back = set(), []
        for s, n, code in zip(seqs, keep, self.codes(seqs)):
            if not code and not 0 <= n <= self.lens[s]:
                code = 71
            if code:
                bad.add(code)
                continue
            back += self.table[s][self.need(n):]
            del self.table[s][self.need(n):]
            self.lens[s] = n
        self.free += reversed(back)
        return bad

    def same(self, p):
        n = int(p.state[0])
        assert p.state.tolist() == [len(self.free), 0]
        assert p.free[:n].tolist() == self.free and p.lens.tolist() == self.lens
        assert p.table.tolist() == [t + [-1] * (self.width - len(t)) for t in self.table]


def ints(values, dev):
    return torch.tensor(values, dtype=torch.int32, device=dev)


def check(got, want, pages=True):
    for name, g, w in zip(got._fields, got, want):
        if name != "pages" or pages:
            assert g.tolist() == w, name


def code(pkg, bad):
    got = pkg.lib.o1_device_error()
    assert (got in bad) if bad else got == 0


@gpu
@pytest.mark.parametrize("pages,page,seqs,width", [(1, 16, 1, 1), (40, 16, 5, 9), (300, 48, 40, 20), (2000, 64, 700, 130), (9000, 16, 1500, 7)])
def test_growing_and_shrinking(pkg, dev, pages, page, seqs, width):
    """Requests of every kind in a row, fitting ones and others, for all sequences and for some in any order."""
    p, m, r = pkg.KvPages(pages, page, seqs, width, dev), Model(pages, page, seqs, width), random.Random(pages)
    m.same(p)
    for step in range(12):
        most = r.choice([1, 1, page, width * page // 3 + 1, width * page + 2])
        names = None if r.random() < 0.3 else r.sample(range(seqs), r.randint(1, seqs))
        batch = seqs if names is None else len(names)
        counts = [r.randint(0, most) for _ in range(batch)]
        if step % 3 == 2:
            counts[r.randrange(batch)] = r.choice([-1, -2 ** 31, 2 ** 31 - 1, width * page + 1])
            if names:
                names[r.randrange(batch)] = r.choice([-1, seqs, 2 ** 31 - 1, -2 ** 31, names[0]])
        total = sum(n for n in counts if 0 <= n <= width * page)
        rows = r.choice([total, total + 5, max(0, total - 3), total // 2])
        want = m.grow(counts, rows, names)
        got = p.grow(ints(counts, dev), rows, None if names is None else ints(names, dev))
        starts = [min(s, 2 ** 30) for s in want[2]]
        check(got, want[:2] + (starts,) + want[3:5], names is not None)
        if names is None:
            assert got.pages.data_ptr() == p.table.data_ptr()
        code(pkg, want[5])
        m.same(p)
        names = None if r.random() < 0.3 else r.sample(range(seqs), r.randint(1, seqs))
        batch = seqs if names is None else len(names)
        keep = [r.choice([0, 0, n, r.randint(0, n)]) for n in (m.lens if names is None else [m.lens[s] for s in names])]
        if step % 3 == 1:
            keep[r.randrange(batch)] = r.choice([-1, 2 ** 31 - 1, -2 ** 31])
            if names:
                names[r.randrange(batch)] = r.choice([-1, seqs, names[0]])
        bad = m.shrink(keep, names)
        p.shrink(ints(keep, dev), None if names is None else ints(names, dev))
        code(pkg, bad)
        m.same(p)
    p.reset()
    Model(pages, page, seqs, width).same(p)


@gpu
@pytest.mark.parametrize("many", [2, 3, 4, 5, 8, 33, 1100])
def test_many_counts_beyond_every_limit(pkg, dev, many):
    """Counts whose sum passes 2^31, and 2^32: none of them is served, nor what is behind them, and what is before them is; sums end at 2^30."""
    seqs = many + 4
    p, m = pkg.KvPages(64, 16, seqs, 8, dev), Model(64, 16, seqs, 8)
    for names in (None, list(range(seqs - 1, -1, -1))):
        counts = [3, 0] + [2 ** 31 - 1] * many + [0, 5]
        got = p.grow(ints(counts, dev), 40, names and ints(names, dev))
        want = m.grow(counts, 40, names)
        check(got, want[:2] + ([min(s, 2 ** 30) for s in want[2]],) + want[3:5], names is not None)
        m.same(p)
        code(pkg, want[5])


@gpu
def test_what_goes_comes_back_in_its_order(pkg, dev):
    p = pkg.KvPages(100, 16, 10, 30, dev)
    p.grow(ints([5, 100, 0, 33], dev), 138, ints([3, 1, 9, 0], dev))
    before = [t.clone() for t in (p.table, p.lens, p.free, p.state)]
    names, old = ints([9, 3, 1, 0], dev), ints([0, 5, 100, 33], dev)
    p.grow(ints([40, 300, 12, 7], dev), 359, names)
    p.shrink(old, names)
    assert all(torch.equal(a, b) for a, b in zip(before, (p.table, p.lens, p.free, p.state)))


@gpu
def test_the_largest_number_of_sequences(pkg, dev):
    seqs, page = 8192, 16
    p, m = pkg.KvPages(20000, page, seqs, 4, dev), Model(20000, page, seqs, 4)
    names = random.Random(1).sample(range(seqs), seqs)
    for counts in ([(7 * i) % 23 for i in range(seqs)], [1] * seqs, [20 + i % 3 for i in range(seqs)]):
        want = m.grow(counts, sum(counts), names)
        check(p.grow(ints(counts, dev), sum(counts), ints(names, dev)), want[:5])
        code(pkg, want[5])
        m.same(p)
    for bad in (names[:5] + names[:1], [0, 0], [5] * 700):
        want = m.grow([1] * len(bad), len(bad), bad)
        check(p.grow(ints([1] * len(bad), dev), len(bad), ints(bad, dev)), want[:5])
        code(pkg, want[5])
    m.same(p)


@gpu
def test_no_pages_left(pkg, dev):
    """Those in front are served, those behind only where they need no page; whatever is refused is as it was."""
    p, m = pkg.KvPages(6, 16, 4, 10, dev), Model(6, 16, 4, 10)
    for counts in ([10, 16, 1, 5], [6, 40, 3, 1], [0, 200, 0, 0], [1, 1, 1, 1]):
        want = m.grow(counts, sum(counts))
        check(p.grow(ints(counts, dev), sum(counts)), want[:4], False)
        code(pkg, want[5])
        m.same(p)


@gpu
@pytest.mark.parametrize("off", [0, 1, 2, 3])
def test_results_at_any_address(pkg, dev, off):
    """The C entry point: results inside larger tensors, tables of a pitch of their own, nothing around them touched."""
    p, m = pkg.KvPages(60, 32, 6, 9, dev), Model(60, 32, 6, 9)
    p.grow(ints([5, 50], dev), 55, ints([2, 4], dev))
    m.grow([5, 50], 55, [2, 4])
    counts, names, rows = [70, 1, 0, 33], [4, 0, 2, 5], 107
    want = m.grow(counts, rows, names)
    slots, positions = torch.full((rows + 8,), 77, dtype=torch.int64, device=dev), torch.full((rows + 8,), 77, dtype=torch.int32, device=dev)
    starts, lens, tables = (torch.full(s, 77, dtype=torch.int32, device=dev) for s in ((5 + 8,), (4 + 8,), (4, 12)))
    on_gpu = ints(names, dev), ints(counts, dev)
    pkg.check(pkg.lib.o1_kv_pages_grow(C.byref(p.c), pkg.ptr(on_gpu[0]), pkg.ptr(on_gpu[1]), 4, pkg.ptr(slots[off:]), pkg.ptr(positions[off:]), rows, pkg.ptr(starts[off:]),
                                       pkg.ptr(lens[off:]), pkg.ptr(tables), 12), "grow")
    for t, w in ((slots, want[0]), (positions, want[1]), (starts, want[2]), (lens, want[3])):
        assert t.tolist() == [77] * off + w + [77] * (len(t) - off - len(w))
    assert tables[:, :9].tolist() == want[4] and (tables[:, 9:] == 77).all()
    m.same(p)


@gpu
def test_captured_requests(pkg, dev):
    """A graph serves what its tensors hold at each replay; rows behind the last one have no slot."""
    p, m = pkg.KvPages(200, 16, 8, 12, dev), Model(200, 16, 8, 12)
    counts, names, keep = ints([3, 4, 5], dev), ints([1, 2, 3], dev), ints([0], dev)
    gone, s = ints([7], dev), torch.cuda.Stream()
    torch.cuda.synchronize()
    try:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=s):
            pkg.use_torch_stream()
            got = p.grow(counts, 64, names)
            p.shrink(keep, gone)
    finally:
        pkg.use_torch_stream()
    for c, n, g in (([3, 4, 5], [1, 2, 3], 7), ([20, 0, 30], [3, 7, 1], 3), ([1, 1, 1], [0, 1, 2], 1), ([60, 40, 2], [4, 5, 6], 0)):
        counts.copy_(ints(c, dev)), names.copy_(ints(n, dev)), gone.copy_(ints([g], dev))
        graph.replay()
        torch.cuda.synchronize()
        want = m.grow(c, 64, n)
        check(got, want[:5])
        m.shrink([0], [g])
        code(pkg, want[5])
        m.same(p)


@gpu
def test_calls_on_another_stream_than_torch_s(pkg, dev):
    """What a call makes is in the order of the library's stream, and lives as long as any part of it."""
    p, m, s = pkg.KvPages(200, 16, 8, 12, dev), Model(200, 16, 8, 12), torch.cuda.Stream()
    counts, names = ints([30, 2, 7], dev), ints([1, 2, 3], dev)
    torch.cuda.synchronize()
    try:
        with torch.cuda.stream(s):
            pkg.use_torch_stream()
        slots, lens = [], []
        for _ in range(20):
            got = p.grow(counts, 39, names)
            slots.append(got.slots), lens.append(got.lens)
            p.shrink(ints([0, 0, 0], dev), names)
            torch.cuda.synchronize()
        del got
        junk = [torch.full((4096,), 77, dtype=torch.int32, device=dev) for _ in range(20)]
    finally:
        pkg.use_torch_stream()
    want = m.grow([30, 2, 7], 39, [1, 2, 3])
    assert all(t.tolist() == want[0] for t in slots) and all(t.tolist() == want[3] for t in lens) and len(junk) == 20


@gpu
def test_arguments_that_do_not_fit(pkg, dev):
    E = pkg.O1Error
    for args in ((0, 16, 1, 1), (4, 24, 2, 2), (4, 16, 9000, 2), (4, 16, 0, 1), (4, 0, 1, 1), (4, 2 ** 24, 1, 2 ** 10)):
        with pytest.raises(E, match="KvPages"):
            pkg.KvPages(*args, device=dev)
    p = pkg.KvPages(8, 16, 4, 3, dev)
    t = (p.table, p.lens, p.free, p.state)
    assert pkg.KvPages.over(*t, 16).pages == 8
    for bad in ((t[0].long(),) + t[1:], (t[0], t[1][:2]) + t[2:], t[:3] + (t[3][:1],), (t[0].T,) + t[1:], (t[0].cpu(),) + t[1:], t[:2] + (t[2][:0],) + t[3:]):
        with pytest.raises(E, match="KvPages"):
            pkg.KvPages.over(*bad, 16)
    one = ints([1], dev)
    for args in ((one.long(), 1), (one.cpu(), 1), (one[None], 1), (ints([1] * 5, dev), 5), (one, -1), (one, 2 ** 30 + 1), (one, 2 ** 31), (ints([1] * 4, dev)[::2], 2), (one, 1, ints([0, 1], dev)),
                 (one, 1, one.long())):
        with pytest.raises(E, match="KvPages.grow"):
            p.grow(*args)
    for args in ((one.long(),), (ints([1] * 5, dev),), (one, ints([0, 1], dev)), (one, one.cpu())):
        with pytest.raises(E, match="KvPages.shrink"):
            p.shrink(*args)
    got = p.grow(one[:0], 3)
    assert got.slots.tolist() == [-1] * 3 and got.starts.tolist() == [0] and got.lens.shape == (0,) and got.pages.shape == (0, 3)
    p.shrink(one[:0])
    assert p.grow(ints([0, 0], dev), 0).slots.shape == (0,)
    Model(8, 16, 4, 3).same(p)
    pkg.check_cuda_errbuf("after refusals")


@gpu
def test_pages_of_another_gpu_are_refused(pkg, dev):
    p = pkg.KvPages(8, 16, 4, 4, dev)
    p._gpu += 1           # (as if its memory were there)
    one = ints([1], dev)
    for call in (p.reset, lambda: p.grow(one, 1), lambda: p.shrink(one)):
        with pytest.raises(pkg.O1Error, match="another GPU than the current one"):
            call()
    p._gpu -= 1
    p.reset()
    check(p.grow(one, 1), ([0], [0], [0, 1], [1], [[0, -1, -1, -1]]))
    code(pkg, set())


def test_entry_points_refuse_before_they_touch_the_gpu(pkg):
    lib, one = pkg.lib, C.c_void_p(4096)
    good = dict(table=4096, lens=4096, free_pages=4096, state=4096, pages=4, page_size=16, max_seqs=3, width=5)

    def call(which, args, **change):
        k = C.byref(pkg.KvPagesC(**{**good, **change}))
        return {"reset": lambda: lib.o1_kv_pages_reset(k), "grow": lambda: lib.o1_kv_pages_grow(k, *args), "shrink": lambda: lib.o1_kv_pages_shrink(k, *args)}[which]()

    grow, shrink = (None, one, 3, one, one, 8, one, one, None, 0), (None, one, 3)
    for which, args in (("reset", ()), ("grow", grow), ("shrink", shrink)):
        for want, change in ((6, dict(table=None)), (6, dict(lens=None)), (6, dict(free_pages=None)), (6, dict(state=None)), (9, dict(pages=0)), (9, dict(page_size=24)), (9, dict(page_size=0)),
                             (9, dict(max_seqs=0)), (9, dict(max_seqs=8193)), (9, dict(width=0)), (9, dict(width=2 ** 28))):
            assert call(which, args, **change) == want, (which, change)
            assert b"kv_pages_" + which.encode() in lib.hd_cuda_last_error()
    for want, at, what in ((6, 1, None), (9, 2, 4), (9, 2, -1), (6, 3, None), (6, 4, None), (9, 5, -1), (6, 6, None), (6, 7, None), (9, 8, one)):
        assert call("grow", grow[:at] + (what,) + grow[at + 1:]) == want, at
    for want, at, what in ((6, 1, None), (9, 2, 4), (9, 2, -1)):
        assert call("shrink", shrink[:at] + (what,) + shrink[at + 1:]) == want, at
    assert call("shrink", (None, None, 0)) == 0 and lib.o1_kv_pages_reset(None) == 6
    lib.hd_cuda_clear_error()


# ------------------------------------------------------------------ together
@gpu
@pytest.mark.parametrize("captured", [False, True])
@pytest.mark.parametrize("kind,layout,page", [("uint4", "half", 64), ("uint4", "interleaved", 16), ("bf16", "half", 32)])
def test_a_server(pkg, dev, kind, layout, page, captured):
    """Prompts come in together, then steps of one row each, one sequence ends and another takes its pages: pages, positions, keys turned, rows kept, attention; each row's
    attention against 64 bits over what is kept.  The steps also as one graph, replayed."""
    heads, kv, seqs = 8, 2, 5
    p = pkg.KvPages(40, page, seqs, 200 // page + 1, dev)
    cache, rope = pkg.KvCache(40, page, kind, kv, dev), pkg.Rotary(128, 128, 10000.0, layout, {"kind": "linear", "factor": 2.0}, dev)
    g = torch.Generator().manual_seed(3)
    held = {}                  # of each sequence: what is kept of its keys and values, (values, magnitudes)

    def keep(s, k, v):
        for i, x in enumerate((k, v)):
            codes = kept(x) if kind == "uint4" else None
            pair = (value(*codes), magnitude(*codes)) if codes else (x.double(), x.double().abs())
            held.setdefault(s, {}).setdefault(i, []).append(pair)

    def rows(n):
        return normal((n, heads + 2 * kv, D), g).to(dev)

    def prompts(names, counts):
        n = sum(counts)
        x = rows(n + 3)                                      # a padded batch: the last rows belong to nobody
        got = p.grow(ints(counts, dev), n + 3, ints(names, dev))
        q, k = rope((x[:, :heads], x[:, heads:heads + kv]), got.positions)
        cache.write(k, x[:, heads + kv:], got.slots)
        k, v, at = k.cpu(), x[:, heads + kv:].cpu(), 0
        for s, c in zip(names, counts):
            held.pop(s, None)
            keep(s, k[at:at + c], v[at:at + c])
            at += c

    names, one, x = ints([3, 0, 4], dev), ints([1, 1, 1], dev), torch.empty(3, heads + 2 * kv, D, dtype=torch.bfloat16, device=dev)

    def step():
        got = p.grow(one, 3, names)
        q, k = rope((x[:, :heads], x[:, heads:heads + kv]), got.positions)
        return q, k, cache.attend(q, got.pages, got.lens, k=k, v=x[:, heads + kv:])

    def check_step(which, q, k, out):
        for i, s in enumerate(which):
            keep(s, k[i:i + 1].cpu(), x[i:i + 1, heads + kv:].cpu())
            (kk, ka), (vv, va) = (tuple(torch.cat(t).repeat_interleave(heads // kv, 1) for t in zip(*held[s][j])) for j in (0, 1))
            qd = q[i].cpu().double()
            z = torch.einsum("hd,thd->ht", qd, kk) / math.sqrt(D)
            size = (torch.einsum("hd,thd->ht", qd.abs(), ka) / math.sqrt(D)).amax(-1)
            pr = torch.softmax(z, -1)
            rel = 2.0 * 2.0 ** -19 * size + 2.0 ** -17 + 2.0 ** -18
            between(out[i], torch.einsum("ht,thd->hd", pr, vv), torch.einsum("ht,thd->hd", pr, va) * rel[:, None] + 1e-30, f"sequence {s}")

    prompts([0, 3, 4, 1], [70, 17, 1, 128])
    graph, s = None, torch.cuda.Stream()
    if captured:
        cache.attend(x[:, :heads], p.table[:3], torch.zeros(3, dtype=torch.int32, device=dev))
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        try:
            with torch.cuda.graph(graph, stream=s):
                pkg.use_torch_stream()
                q, k, out = step()
        finally:
            pkg.use_torch_stream()
    for which in ([3, 0, 4], [3, 0, 4], [1, 3, 0], [4, 1, 3]):
        names.copy_(ints(which, dev)), x.copy_(rows(3))
        if graph:
            graph.replay()
        else:
            q, k, out = step()
        torch.cuda.synchronize()
        check_step(which, q, k, out)
    p.shrink(ints([0, 0], dev), ints([1, 4], dev))
    prompts([2, 4], [90, 33])
    for which in ([2, 4, 0], [3, 2, 4]):
        names.copy_(ints(which, dev)), x.copy_(rows(3))
        if graph:
            graph.replay()
        else:
            q, k, out = step()
        torch.cuda.synchronize()
        check_step(which, q, k, out)
    assert pkg.lib.o1_device_error() == 0


def test_results_over_what_is_read_are_refused(pkg):
    """Results that share a byte with one another, with the requests or with the pages' own arrays: other blocks still read those.  (All of these are refused before anything is launched.)"""
    base = dict(table=0x100000, lens=0x200000, free_pages=0x300000, state=0x400000)
    k = pkg.KvPagesC(**base, pages=50, page_size=16, max_seqs=8, width=5)
    good = dict(seqs=0x500000, counts=0x600000, slots=0x700000, positions=0x800000, starts=0x900000, lens=0xA00000, tables=0xB00000)
    size = dict(seqs=5 * 4, counts=5 * 4, slots=11 * 8, positions=11 * 4, starts=6 * 4, lens=5 * 4, tables=(4 * 7 + 5) * 4)
    own = dict(table=8 * 5 * 4, lens=8 * 4, free_pages=50 * 4, state=8)
    for name in ("slots", "positions", "starts", "lens", "tables"):
        others = [(good[o], size[o]) for o in good if o != name] + [(base[o], own[o]) for o in own]
        for at, n in others:
            for where in (at, at + n - 4, at - size[name] + 4):
                p = {o: C.c_void_p(v) for o, v in {**good, name: where}.items()}
                assert pkg.lib.o1_kv_pages_grow(C.byref(k), p["seqs"], p["counts"], 5, p["slots"], p["positions"], 11, p["starts"], p["lens"], p["tables"], 7) == 9, (name, hex(where))
                assert b"shares memory" in pkg.lib.hd_cuda_last_error()
    pkg.lib.hd_cuda_clear_error()


@gpu
def test_results_right_behind_one_another(pkg, dev):
    """One buffer for all results and the requests, not a byte between them."""
    p, m = pkg.KvPages(60, 16, 6, 9, dev), Model(60, 16, 6, 9)
    counts, names, rows = [70, 1, 0, 33], [4, 0, 2, 5], 104
    want = m.grow(counts, rows, names)
    sizes = [rows * 2, rows, 5, 4, 4 * 9, 4, 4]
    buf = torch.full((sum(sizes),), 77, dtype=torch.int32, device=dev)
    slots, positions, starts, lens, tables, c, n = buf.split(sizes)
    c.copy_(ints(counts, dev)), n.copy_(ints(names, dev))
    pkg.check(pkg.lib.o1_kv_pages_grow(C.byref(p.c), pkg.ptr(n), pkg.ptr(c), 4, pkg.ptr(slots), pkg.ptr(positions), rows, pkg.ptr(starts), pkg.ptr(lens), pkg.ptr(tables), 9), "grow")
    check(pkg.kvcache.Grown(slots.view(torch.int64), positions, starts, lens, tables.view(4, 9)), want[:5])
    assert c.tolist() == counts and n.tolist() == names
    m.same(p)
