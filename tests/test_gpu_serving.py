"""The decoder blocks over rows of four bits, and with pages that are handed out on the GPU.

Bound for rows of four bits: the blocks' own tolerance is 1e-2 a block (2-norm), e.  Values that differ by e take another code where a midpoint lies between, in a
share of about 0.8 e / 0.36 of them (16 codes over the 5.4 deviations that 128 normal values spread), and are then 0.36 deviations apart: 0.36 sqrt(2.2 e) = 0.53 sqrt(e).  Half as
much again for the grid, which moves with a row's least and largest value: 0.8 sqrt(e)."""
import ctypes as C
import math

import pytest
import torch

import test_gpu_decode as dec_tests
import test_gpu_uint4 as four
from test_gpu_decode import DIMS, ids_of, models, reference  # noqa: F401

gpu = pytest.mark.gpu


def within(got, want, tol):
    got, want = got.cpu().double(), want.double()
    rel = float((got - want).norm() / want.norm())
    assert rel <= tol, f"relative L2 {rel:.3g}, not {tol:.3g}"


@gpu
@pytest.mark.parametrize("layers", [1, 3])
@pytest.mark.parametrize("lens,page", [([1], 16), ([5, 40, 130], 64), ([16, 17, 15, 64, 1, 2, 3, 33, 200], 32)])
def test_prompts_and_the_rows_after_them(pkg, dev, models, monkeypatch, layers, lens, page):  # noqa: F811
    monkeypatch.setattr(dec_tests, "quantised", four.quantised)
    monkeypatch.setattr(dec_tests, "value", four.value)
    steps, weights = 5, models[layers]
    seqs = [ids_of(n + steps, 10 * n + i) for i, n in enumerate(lens)]
    dec = pkg.Decoder(weights, len(lens), max(lens) + steps, "uint4", page)
    wants = [reference(weights, s, n, "uint4") for s, n in zip(seqs, lens)]
    names = [dec.prompt(s[:n].to(dev))[0] for s, n in zip(seqs, lens)]
    for i in range(steps):
        rows = dec.step(names, torch.tensor([int(s[n + i]) for s, n in zip(seqs, lens)]).to(dev))
        within(rows, torch.stack([want[0][n + i] for n, want in zip(lens, wants)]), 0.8 * math.sqrt(1e-2 * layers))
    for name, want in zip(names, wants):
        for layer in range(layers):
            for got, kept in zip(dec.rows(name, layer), want[1][layer]):
                within(got, kept, 0.8 * math.sqrt(1e-2 * (layer + 1)))
    assert pkg.lib.o1_device_error() == 0


@gpu
@pytest.mark.parametrize("kind", ["bf16", "uint4"])
def test_a_captured_step_with_pages_of_the_gpu(pkg, dev, models, kind):  # noqa: F811
    """o1_decode_step in a graph, with lengths and pages from KvPages: replayed, it gives the rows that Decoder.step gives, for sequences that change from replay to replay."""
    w, n, page, layers = models[3], 3, 16, 3
    lens = [9, 40, 17, 1]
    prompts = [ids_of(k, k) for k in lens]
    plain = pkg.Decoder(w, len(lens), 64, kind, page)
    names = [plain.prompt(p.to(dev))[0] for p in prompts]

    dec = pkg.Decoder(w, len(lens), 64, kind, page)                # its caches and scratch, with pages of the GPU's own
    pool = pkg.KvPages(16, page, len(lens), 4, dev)
    d = dec.dims
    for i, p in enumerate(prompts):
        got = pool.grow(torch.tensor([len(p)], dtype=torch.int32, device=dev), len(p), torch.tensor([i], dtype=torch.int32, device=dev))
        ids, pos = p.to(dev), got.positions.float().expand(3, -1).contiguous()
        out, s = torch.empty(len(p), DIMS["hidden"], dtype=torch.bfloat16, device=dev), dec._room(len(p))
        pkg.check(pkg.lib.o1_prompt_rows(C.byref(w.binding), dec._c, pkg.ptr(ids), pkg.ptr(pos), pkg.ptr(got.slots), pkg.ptr(s), s.numel(), pkg.ptr(out), len(p), *d), "o1_prompt_rows")
    ids, which, ones = torch.zeros(n, dtype=torch.int64, device=dev), torch.zeros(n, dtype=torch.int32, device=dev), torch.ones(n, dtype=torch.int32, device=dev)
    out, scratch = torch.empty(n, DIMS["hidden"], dtype=torch.bfloat16, device=dev), torch.zeros(pkg.lib.o1_decode_scratch_bytes(n, *d[:5]), dtype=torch.uint8, device=dev)

    def step():
        got = pool.grow(ones, n, which)
        pos = got.positions.float().expand(3, n).contiguous()
        pkg.check(pkg.lib.o1_decode_step(C.byref(w.binding), dec._c, pkg.ptr(ids), pkg.ptr(pos), pkg.ptr(got.pages), 4, 4, pkg.ptr(got.lens), pkg.ptr(scratch), scratch.numel(),
                                         pkg.ptr(out), n, *d), "o1_decode_step")
        return got, pos

    torch.cuda.synchronize()
    graph, stream = torch.cuda.CUDAGraph(), torch.cuda.Stream()
    try:
        with torch.cuda.graph(graph, stream=stream):
            pkg.use_torch_stream()
            kept = step()
    finally:
        pkg.use_torch_stream()
    for i, seqs in enumerate(([0, 1, 2], [3, 1, 0], [2, 3, 1], [2, 3, 1])):
        new = ids_of(n, 70 + i).to(dev)
        want = plain.step([names[s] for s in seqs], new)
        ids.copy_(new), which.copy_(torch.tensor(seqs, dtype=torch.int32))
        graph.replay()
        torch.cuda.synchronize()
        assert kept[0].lens.tolist() == [plain._len[names[s]] for s in seqs]
        assert torch.equal(out, want)
    assert pkg.lib.o1_device_error() == 0


@gpu
def test_a_step_in_either_scratch(pkg, dev, models):  # noqa: F811
    """o1_decode_step over rows of four bits of many sequences, in the scratch that any kind needs and in that of four bits: the rows that Decoder.step gives, within a block's tolerance of them."""
    w, n, page, layers = models[3], 80, 16, 3
    lens = [1 + (37 * i) % 150 for i in range(n)]
    dec = pkg.Decoder(w, n, 160, "uint4", page)
    names = [dec.prompt(ids_of(k, k).to(dev))[0] for k in lens]
    for s, k in zip(names, lens):
        dec._grow(s, k + 1)             # the new row's page
    ids = ids_of(n, 5).to(dev)
    tables = torch.stack([dec._table[s] for s in names])
    at = torch.tensor(lens, dtype=torch.int32, device=dev) + 1
    pos = (at - 1).float().expand(3, n).contiguous()
    outs = []
    for kind in (0, 4):
        size = pkg.lib.o1_decode_scratch_bytes_of(kind, n, *dec.dims[:5])
        scratch = torch.full((size + 4096,), 0xA5, dtype=torch.uint8, device=dev)
        scratch[:32768 + 256] = 0
        out = torch.empty(n, DIMS["hidden"], dtype=torch.bfloat16, device=dev)
        for _ in range(2):          # (the row is written again)
            pkg.check(pkg.lib.o1_decode_step(C.byref(w.binding), dec._c, pkg.ptr(ids), pkg.ptr(pos), pkg.ptr(tables), dec.width, dec.width, pkg.ptr(at), pkg.ptr(scratch), size, pkg.ptr(out), n,
                                             *dec.dims), "o1_decode_step")
        assert (scratch[size:] == 0xA5).all()
        outs.append(out)
    want = dec.step(names, ids)
    assert torch.equal(outs[1], want)
    within(outs[0], want.cpu(), 0.8 * math.sqrt(1e-2 * layers))
