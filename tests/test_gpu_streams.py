"""Calls whose library stream is not torch's current one: caches, results and tables are made in the order of the library's."""
import ctypes as C
import math

import pytest
import torch

from test_gpu_decode import ids_of, models, weights  # noqa: F401
from test_gpu_kvcache import Case, D, gen, normal

gpu = pytest.mark.gpu


class Apart:
    """The library on a stream of its own, torch's current one busy."""

    def __init__(self, pkg, cycles=300000000):
        self.pkg, self.cycles = pkg, cycles

    def __enter__(self):
        torch.cuda.synchronize()
        self.s = torch.cuda.Stream()
        self.pkg.lib.o1_set_stream(C.c_void_p(self.s.cuda_stream))
        torch.cuda._sleep(self.cycles)
        return self.s

    def __exit__(self, *a):
        torch.cuda.synchronize()
        self.pkg.use_torch_stream()


@gpu
def test_shared_vectors_on_another_stream(pkg, dev):
    """One gate for both groups is copied for the call: where the call reads it, and not into memory that is taken back before."""
    x, b, w = normal((6, 4096), gen(1)).to(dev), normal((6, 4096), gen(2)).to(dev), normal((4096,), gen(3)).to(dev)
    gate, m2 = normal((4096,), gen(4)).to(dev), normal((2, 4096), gen(5)).to(dev)
    want = pkg.residual_norm(x, b, w, gate=gate, scale=m2, shift=m2)
    t = [torch.full((2, 4096), math.nan, dtype=torch.bfloat16, device=dev) for _ in range(8)]
    y, h = torch.empty_like(x), torch.empty_like(x)
    del t
    with Apart(pkg):
        pkg.residual_norm(x, b, w, gate=gate, scale=m2, shift=m2, y=y, h=h)
    assert torch.equal(y, want[0]) and torch.equal(h, want[1])


@gpu
@pytest.mark.parametrize("what", ["norm", "read", "attend"])
def test_results_on_another_stream(pkg, dev, what):
    """Results do not lie in memory that torch's stream has yet to finish with."""
    c = Case(pkg, dev, "bf16", [40, 20], 2, 16)
    c.fill()
    q = normal((2, 4, D), gen(1)).to(dev)
    x, w = normal((64, 2048), gen(1)).to(dev), normal((2048,), gen(3)).to(dev)
    slots = c.slots(0).to(dev)
    call = {"norm": lambda: pkg.residual_norm(x, x, w), "read": lambda: c.cache.read(slots),
            "attend": lambda: c.cache.attend(q, c.dtable, c.dlens, lse=True)}[what]
    want = [t.clone() for t in call()]
    with Apart(pkg):
        call()          # a stream's workspace
    with Apart(pkg):
        old = [torch.empty_like(t).fill_(9.0) for t in want for _ in range(6)]
        del old
        got = call()
    assert all(torch.equal(a, b) for a, b in zip(got, want))


@gpu
def test_a_cache_made_on_another_stream(pkg, dev):
    """Its zeros come before its rows."""
    x = normal((20, 2, D), gen(1)).to(dev)
    slots = torch.arange(20, device=dev)
    with Apart(pkg):
        cache = pkg.KvCache(4, 16, "int8", 2, dev)
        cache.write(x, x, slots)
    assert (cache.read(slots)[0] != 0).any()


@gpu
def test_decoder_on_another_stream(pkg, dev, weights):
    prompts, new = [ids_of(n, n).to(dev) for n in (40, 7)], [ids_of(2, 5 + i).to(dev) for i in range(3)]

    def run(dec):
        got, names = [], []
        for p in prompts:
            name, rows = dec.prompt(p)
            names.append(name)
            got.append(rows)
        for ids in new:
            got.append(dec.step(names, ids))
        return got + list(dec.rows(names[0], 1))
    want = run(pkg.Decoder(weights, 2, 64, "int8", 16))
    torch.cuda.synchronize()
    junk = [torch.randint(0, 2 ** 30, (n,), device=dev) for n in (2, 64, 512, 4096, 65536) for _ in range(8)]
    torch.cuda.synchronize()
    del junk
    with Apart(pkg):
        got = run(pkg.Decoder(weights, 2, 64, "int8", 16))
    assert pkg.lib.o1_device_error() == 0
    assert all(torch.equal(a, b) for a, b in zip(got, want))


@gpu
def test_what_is_filled_for_the_default_stream(pkg, dev):
    """The library on the default stream, torch on another: workspaces are filled on the default stream, not on a third one."""
    import sys
    kv = sys.modules[pkg.KvCache.__module__]
    try:
        for s in (torch.cuda.default_stream(), torch.cuda.Stream()):
            pkg.lib.o1_set_stream(C.c_void_p(s.cuda_stream))
            with torch.cuda.stream(torch.cuda.Stream()), kv._on_library(dev):
                assert torch.cuda.current_stream().cuda_stream == s.cuda_stream
    finally:
        pkg.use_torch_stream()


@gpu
def test_an_engine_on_another_stream(pkg, dev):
    """The timestep of a forward and of a guided step is set where they read it."""
    T, I = 19, 48
    w = pkg.Weights(n_layers=1, seed=3, device=dev)
    eng = pkg.Engine(w, T, I)
    pos, _ = pkg.seq_t2i(T, 6, 8)
    pos, ids = pos.to(dev), ids_of(T, 1).to(dev)
    ids[-1] = 151673      # the row of the timestep
    z = normal((I, 3072), gen(1)).to(dev)

    def run():
        return eng.forward(ids, pos, z, 0.3), eng.denoise_step_cfg(ids, ids, pos, z, 0.7, 0.6, 2.0), \
            eng.denoise_step_cfg_branches((ids, pos, T - 1), (ids, pos, T - 1), z, 0.5, 0.4, 2.0)
    want = [t.clone() for t in run()]
    assert not torch.equal(eng.forward(ids, pos, z, 0.9), want[0])
    for i in range(3):
        eng.forward(ids, pos, z, 0.9)
        with Apart(pkg):
            old = [torch.full_like(t, 9.0) for t in want for _ in range(4)]
            del old
            got = run()[i]
        assert torch.equal(got, want[i])
