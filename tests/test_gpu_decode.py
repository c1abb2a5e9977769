"""Prompts and the rows after them over cached keys and values: Decoder (o1_prompt_rows, o1_decode_step) against the whole sequence, computed in 64 bits
between the points where the decoder stores bf16 (as the oracle does), within the framework's tolerance of a block for each block (cosine >= 0.999,
relative L2 <= 1e-2; single roundings that fall the other way make the rest of a chain differ, so blocks add)."""
import ctypes as C
import math

import pytest
import torch

from test_gpu_kvcache import quantised, value

gpu = pytest.mark.gpu
DIMS = dict(hidden=512, heads=4, kv_heads=2, head_dim=128, ff=1024, vocab=1000)
SECTION = [24, 20, 20]


@pytest.fixture(scope="module")
def models(pkg):
    if not torch.cuda.is_available():
        pytest.skip("no CUDA device")
    pkg.use_torch_stream()
    return {n: pkg.Weights(n_layers=n, seed=5, weight_set="B", device="cuda:0", std=0.05, **DIMS) for n in (1, 3)}


@pytest.fixture
def weights(models):
    return models[3]


def r(x):
    return x.to(torch.bfloat16).double()


def reference(w, ids, prompt, kind):
    """Rows behind the final norm of a text sequence, and each layer's keys and values as they are kept.  Rows from `prompt` on attend to those."""
    d = w.dims

    def t(layer, name):
        return w.tensor(layer, name).cpu().double()

    def norm(a, v):
        return r(a / torch.sqrt((a * a).mean(-1, keepdim=True) + 1e-6) * v)

    n = ids.numel()
    half = d["head_dim"] // 2
    freq = 5000000.0 ** (-torch.arange(half, dtype=torch.float64) * 2 / d["head_dim"])
    ang = torch.arange(n, dtype=torch.float64)[:, None] * freq      # text rows have the same position on all three axes
    cos, sin = (torch.cat([f(ang), f(ang)], 1)[:, None, :] for f in (torch.cos, torch.sin))

    def rope(x):
        turned = torch.cat([-x[..., half:], x[..., :half]], -1)
        return r(r(x * cos) + r(turned * sin))

    x = t(-1, "embed_tokens")[ids.cpu()]
    mask = torch.full((n, n), -math.inf, dtype=torch.float64).triu(1)
    kept = []
    h = norm(x, t(0, "input_ln"))
    for layer in range(w.n_layers):
        q, k, v = (r(h @ t(layer, name).T).view(n, -1, d["head_dim"]) for name in ("q_proj", "k_proj", "v_proj"))
        q, k = rope(norm(q, t(layer, "q_norm"))), rope(norm(k, t(layer, "k_norm")))
        kept.append(tuple(value(*quantised(x_.to(torch.bfloat16), kind)) for x_ in (k, v)))
        g = d["heads"] // d["kv_heads"]
        parts = []
        for rows, (k_, v_) in ((slice(0, prompt), (k, v)), (slice(prompt, n), kept[-1])):
            z = torch.einsum("qhd,khd->hqk", q[rows], k_.repeat_interleave(g, 1)) / math.sqrt(d["head_dim"]) + mask[rows]
            parts.append(torch.einsum("hqk,khd->qhd", torch.softmax(z, -1), v_.repeat_interleave(g, 1)).reshape(-1, g * d["kv_heads"] * d["head_dim"]))
        a = r(torch.cat(parts))
        y = x + r(a @ t(layer, "o_proj").T)
        x, h = r(y), norm(y, t(layer, "post_ln"))
        gate, up = r(h @ t(layer, "gate_proj").T), r(h @ t(layer, "up_proj").T)
        y = x + r(r(r(gate * torch.sigmoid(gate)) * up) @ t(layer, "down_proj").T)
        x, h = r(y), norm(y, t(layer + 1, "input_ln") if layer + 1 < w.n_layers else t(-1, "fnorm_w"))
    return h, kept


def near(got, want, tol):
    got, want = got.cpu().double(), want.double()
    rel = (got - want).norm() / want.norm()
    cos = (got * want).sum() / (got.norm() * want.norm())
    assert cos >= 0.999 and rel <= tol, f"cosine {cos:.6f}, relative L2 {rel:.3g}"


def ids_of(n, seed):
    return torch.randint(0, DIMS["vocab"], (n,), generator=torch.Generator().manual_seed(seed))


@gpu
@pytest.mark.parametrize("layers", [1, 3])
@pytest.mark.parametrize("kind,tol", [("bf16", 1e-2), ("fp8", 5e-2), ("int8", 1e-2)])
@pytest.mark.parametrize("lens,page", [([1], 16), ([5, 40, 130], 64), ([16, 17, 15, 64, 1, 2, 3, 33, 200], 16)])
def test_prompts_and_the_rows_after_them(pkg, dev, models, layers, kind, tol, lens, page):
    """Every step's rows beside the whole sequence's.  (A key that differs in its last bit can take another code, and e4m3's lie 2^-3 apart: its bound is wider.)"""
    steps, weights = 5, models[layers]
    seqs = [ids_of(n + steps, 10 * n + i) for i, n in enumerate(lens)]
    dec = pkg.Decoder(weights, len(lens), max(lens) + steps, kind, page)
    wants = [reference(weights, s, n, kind) for s, n in zip(seqs, lens)]
    names = []
    for s, n, want in zip(seqs, lens, wants):
        name, rows = dec.prompt(s[:n].to(dev))
        near(rows, want[0][:n], 1e-2 * layers)
        names.append(name)
    for i in range(steps):
        new = torch.tensor([int(s[n + i]) for s, n in zip(seqs, lens)]).to(dev)
        rows = dec.step(names, new)
        near(rows, torch.stack([want[0][n + i] for n, want in zip(lens, wants)]), tol * layers)
    for name, want in zip(names, wants):
        for layer in range(layers):
            k, v = dec.rows(name, layer)
            near(k, want[1][layer][0], tol * (layer + 1))
            near(v, want[1][layer][1], tol * (layer + 1))


@gpu
def test_a_row_does_not_depend_on_the_others(pkg, dev, weights):
    """A sequence alone and among others: the same bits; pages of a closed sequence are used again."""
    prompts = [ids_of(n, n) for n in (20, 300, 7, 64)]
    a, b = pkg.Decoder(weights, 4, 320, "int8", 32), pkg.Decoder(weights, 1, 320, "int8", 32)
    names = [a.prompt(p.to(dev))[0] for p in prompts]
    a.close(names[1])
    again, _ = a.prompt(prompts[1].to(dev))
    names[1] = again
    alone, _ = b.prompt(prompts[2].to(dev))
    for i in range(4):
        new = ids_of(4, 50 + i).to(dev)
        together = a.step(names, new)
        assert torch.equal(together[2:3], b.step([alone], new[2:3]))
    assert torch.equal(a.rows(names[2], 1)[0], b.rows(alone, 1)[0])


@gpu
def test_arguments_that_do_not_fit(pkg, dev, weights):
    dec = pkg.Decoder(weights, 2, 32, "bf16", 16)
    E = pkg.O1Error
    for bad in (torch.zeros(3, dtype=torch.int32, device=dev), torch.zeros(0, dtype=torch.int64, device=dev), torch.zeros(3, dtype=torch.int64), torch.zeros(1, 3, dtype=torch.int64, device=dev)):
        with pytest.raises(E, match="Decoder.prompt"):
            dec.prompt(bad)
    with pytest.raises(E, match="max_tokens"):
        dec.prompt(ids_of(33, 1).to(dev))
    a, _ = dec.prompt(ids_of(32, 1).to(dev))
    b, _ = dec.prompt(ids_of(3, 1).to(dev))
    with pytest.raises(E, match="2 sequences are open"):
        dec.prompt(ids_of(3, 1).to(dev))
    with pytest.raises(E, match="max_tokens"):
        dec.step([a], ids_of(1, 1).to(dev))
    with pytest.raises(E, match="different"):
        dec.step([b, b], ids_of(2, 1).to(dev))
    with pytest.raises(E, match="no sequence"):
        dec.step([77], ids_of(1, 1).to(dev))
    assert dec.step([], torch.zeros(0, dtype=torch.int64, device=dev)).shape == (0, DIMS["hidden"])
    dec.close(a)
    dec.prompt(ids_of(32, 2).to(dev))


def test_entry_points_refuse_before_they_touch_the_gpu(pkg):
    lib = pkg.lib
    one = C.c_void_p(4096)
    blocks = (pkg.BlockBinding * 1)()
    bw = pkg.ForwardBinding(embed_tokens=4096, fnorm_w=4096, n_layers=1, blocks=C.cast(blocks, C.POINTER(pkg.BlockBinding)))
    cache = (pkg.KvCacheC * 1)(pkg.KvCacheC(4096, 4096, None, None, 0, 4, 16, 2, 128))
    need = lib.o1_decode_scratch_bytes(3, 4, 2, 512, 1024, 128)
    assert need > 0 and lib.o1_decode_scratch_bytes(3, 4, 3, 512, 1024, 128) == -1
    # up to eight rows take the same room, beyond that it grows with the rows
    assert lib.o1_decode_scratch_bytes(8, 4, 2, 512, 1024, 128) == need < lib.o1_decode_scratch_bytes(9, 4, 2, 512, 1024, 128)

    def step(bw_=bw, caches=cache, ids=one, pos=one, pages=one, lens=one, ws=one, nb=need, out=one, batch=3, heads=4, kv=2, hidden=512, ff=1024, hd=128):
        return lib.o1_decode_step(C.byref(bw_), caches, ids, pos, pages, 4, 4, lens, ws, nb, out, batch, heads, kv, hidden, ff, hd, 1000)

    def prompt(ids=one, pos=one, slots=one, ws=one, nb=need, out=one, rows=3, hidden=512):
        return lib.o1_prompt_rows(C.byref(bw), cache, ids, pos, slots, ws, nb, out, rows, 4, 2, hidden, 1024, 128, 1000)

    for want, args in ((6, dict(caches=None)), (6, dict(ids=None)), (6, dict(pos=None)), (6, dict(pages=None)), (6, dict(lens=None)), (6, dict(ws=None)), (6, dict(out=None)),
                       (6, dict(bw_=pkg.ForwardBinding())), (7, dict(nb=need - 1)), (9, dict(batch=-1)), (9, dict(heads=3)), (9, dict(hidden=500)), (9, dict(ff=100)), (9, dict(hd=64)),
                       (5, dict(heads=4, kv=1))):
        assert step(**args) == want, args
        assert b"decode" in lib.hd_last_error(), args
    for want, args in ((6, dict(ids=None)), (6, dict(slots=None)), (6, dict(out=None)), (7, dict(nb=5)), (9, dict(rows=-1)), (9, dict(hidden=511))):
        assert prompt(**args) == want, args
    assert step(batch=0) == 0 and prompt(rows=0) == 0
    lib.hd_cuda_clear_error()


def raw_step(pkg, dec, names, ids, pages, lens):
    """Decoder.step's call with tables of the test's own."""
    n = len(names)
    pos = (lens - 1).clamp(0, 10 ** 6).float().expand(3, n).contiguous()
    out = torch.full((n, dec.dims[2]), 7.0, dtype=torch.bfloat16, device=dec.device)
    s = dec._room(n)
    pkg.check(pkg.lib.o1_decode_step(C.byref(dec.w.binding), dec._c, pkg.ptr(ids), pkg.ptr(pos), pkg.ptr(pages), pages.size(1), pages.size(1), pkg.ptr(lens),
                                     pkg.ptr(s), s.numel(), pkg.ptr(out), n, *dec.dims), "o1_decode_step")
    return out


@gpu
@pytest.mark.parametrize("what,code", [("page", 70), ("negative", 70), ("length", 71), ("long", 71)])
@pytest.mark.parametrize("kind", ["bf16", "fp8"])
def test_a_wrong_entry_reaches_one_sequence_only(pkg, dev, weights, kind, what, code):
    """A page or length of one sequence that does not fit: the others' rows, and what every layer keeps of them, are as without it."""
    lens = [9, 5, 14]
    dec = pkg.Decoder(weights, 3, 64, kind, 16)
    names = [dec.prompt(ids_of(n, n).to(dev))[0] for n in lens]
    before = [[t.clone() for t in (c.k.view(torch.uint8), c.v.view(torch.uint8))] for c in dec.caches]
    ids = ids_of(3, 99).to(dev)
    pages = torch.stack([dec._table[s] for s in names])
    ln = torch.tensor([n + 1 for n in lens], dtype=torch.int32, device=dev)
    want = raw_step(pkg, dec, names, ids, pages, ln)
    after = [[t.clone() for t in (c.k.view(torch.uint8), c.v.view(torch.uint8))] for c in dec.caches]
    for c, (k, v) in zip(dec.caches, before):
        c.k.view(torch.uint8).copy_(k), c.v.view(torch.uint8).copy_(v)
    bad_pages, bad_ln = pages.clone(), ln.clone()
    if what == "page":
        bad_pages[1, 0] = dec.caches[0].pages
    elif what == "negative":
        bad_pages[1, 0] = -3
    else:
        bad_ln[1] = -1 if what == "length" else 16 * pages.size(1) + 1
    got = raw_step(pkg, dec, names, ids, bad_pages, bad_ln)
    assert pkg.lib.o1_device_error() == code and pkg.lib.o1_device_error() == 0
    assert torch.equal(got[[0, 2]], want[[0, 2]])
    mine = {int(p) for p in pages[1]}
    others = [p for p in range(dec.caches[0].pages) if p not in mine]
    for c, (k, v) in zip(dec.caches, after):
        assert torch.equal(c.k.view(torch.uint8)[others], k[others]) and torch.equal(c.v.view(torch.uint8)[others], v[others])


@gpu
def test_a_step_does_not_wait(pkg, dev, weights):
    """A prompt and a step return while the stream is still busy with what came before."""
    dec = pkg.Decoder(weights, 2, 64, "int8", 16)
    a, _ = dec.prompt(ids_of(20, 1).to(dev))
    new, two = ids_of(1, 2).to(dev), ids_of(9, 3).to(dev)
    dec.step([a], new)
    b, _ = dec.prompt(two)
    dec.close(b)
    for call in (lambda: dec.step([a], new), lambda: dec.prompt(two)):
        torch.cuda.synchronize()
        torch.cuda._sleep(2000000000)
        e = torch.cuda.Event()
        e.record()
        call()
        assert not e.query()
    torch.cuda.synchronize()


@gpu
def test_calls_in_a_capture_are_refused(pkg, dev, weights):
    """A graph would keep the lengths and pages of its capture; nothing is changed, and what else is captured stays."""
    dec = pkg.Decoder(weights, 2, 64, "bf16", 16)
    a, _ = dec.prompt(ids_of(20, 1).to(dev))
    new, x = ids_of(1, 2).to(dev), torch.zeros(4, device=dev)
    s = torch.cuda.Stream()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    try:
        with torch.cuda.graph(graph, stream=s):
            pkg.use_torch_stream()
            x += 1
            with pytest.raises(pkg.O1Error, match="Decoder.step.*graph"):
                dec.step([a], new)
            with pytest.raises(pkg.O1Error, match="Decoder.prompt.*graph"):
                dec.prompt(new)
    finally:
        pkg.use_torch_stream()
    graph.replay()
    assert (x == 1).all() and dec.rows(a, 0)[0].size(0) == 20
    dec.step([a], new)


class Fails:
    """The library with one entry point that fails."""

    def __init__(self, lib, name):
        self._lib, self._name = lib, name

    def __getattr__(self, n):
        return (lambda *a: 3) if n == self._name else getattr(self._lib, n)


@gpu
def test_failed_calls_change_nothing(pkg, dev, weights, monkeypatch):
    """A failed prompt leaves no sequence open, a failed step counts no row."""
    import sys
    kv = sys.modules[pkg.Decoder.__module__]
    dec, same = pkg.Decoder(weights, 2, 64, "bf16", 16), pkg.Decoder(weights, 2, 64, "bf16", 16)
    a, _ = dec.prompt(ids_of(20, 1).to(dev))
    b, _ = same.prompt(ids_of(20, 1).to(dev))
    free = len(dec._free)
    with monkeypatch.context() as m:
        m.setattr(kv, "lib", Fails(kv.lib, "o1_prompt_rows"))
        for _ in range(3):
            with pytest.raises(pkg.O1Error, match="o1_prompt_rows"):
                dec.prompt(ids_of(30, 2).to(dev))
    assert len(dec._free) == free
    c, _ = dec.prompt(ids_of(30, 2).to(dev))
    with monkeypatch.context() as m:
        m.setattr(kv, "lib", Fails(kv.lib, "o1_decode_step"))
        with pytest.raises(pkg.O1Error, match="o1_decode_step"):
            dec.step([a, c], ids_of(2, 3).to(dev))
    new = ids_of(1, 4).to(dev)
    assert torch.equal(dec.step([a], new), same.step([b], new))
    assert dec.rows(a, 0)[0].size(0) == 21


class Kept:
    """Weights whose tensors are brought to the host, in 64 bits, once."""

    def __init__(self, w):
        self.w, self.dims, self.n_layers, self.got = w, w.dims, w.n_layers, {}

    def tensor(self, layer, name):
        if (layer, name) not in self.got:
            self.got[layer, name] = self.w.tensor(layer, name).cpu().double()
        return self.got[layer, name]


@gpu
@pytest.mark.parametrize("kind,tol", [("bf16", 1e-2), ("fp8", 5e-2), ("int8", 1e-2)])
@pytest.mark.parametrize("size,count", [("small", 33), ("small", 140), ("full", 12)])
def test_steps_of_many_rows(pkg, dev, models, kind, tol, size, count):
    """More rows than the few that a step's products take as eight, and a block of the framework's own size: 32 / 8 heads, width 4096, 12288 in the middle."""
    w = models[1] if size == "small" else pkg.Weights(n_layers=1, seed=6, weight_set="B", device="cuda:0")
    kept, steps = Kept(w), 2
    lens = [1 + (29 * i) % 71 for i in range(count)]
    seqs = [ids_of(n + steps, 100 * n + i) for i, n in enumerate(lens)]
    dec = pkg.Decoder(w, count, max(lens) + steps, kind, 16)
    names = [dec.prompt(s[:n].to(dev))[0] for s, n in zip(seqs, lens)]
    some = range(0, count, max(1, count // 12))
    wants = {i: reference(kept, seqs[i], lens[i], kind)[0] for i in some}
    for at in range(steps):
        rows = dec.step(names, torch.tensor([int(s[n + at]) for s, n in zip(seqs, lens)]).to(dev))
        near(rows[list(some)], torch.stack([wants[i][lens[i] + at] for i in some]), tol)
    assert pkg.lib.o1_device_error() == 0


@gpu
@pytest.mark.parametrize("layers", [1, 3])
def test_steps_beside_the_prompt_pass(pkg, dev, models, layers):
    """Rows that were steps, beside the same rows in one prompt pass: each is within the tolerance of the reference, so they are within twice that of one another."""
    dec = pkg.Decoder(models[layers], 4, 400, "bf16", 32)
    for n, steps in ((1, 6), (30, 5), (300, 9)):
        ids = ids_of(n + steps, n).to(dev)
        name, _ = dec.prompt(ids[:n])
        got = torch.cat([dec.step([name], ids[n + i:n + i + 1]) for i in range(steps)])
        whole, rows = dec.prompt(ids)
        near(got, rows[n:].cpu(), 2e-2 * layers)
        for layer in range(layers):
            for a, b in zip(dec.rows(name, layer), dec.rows(whole, layer)):
                near(a, b.cpu(), 2e-2 * (layer + 1))
        dec.close(name)
        dec.close(whole)
