"""Rotary positions (Rotary, o1_rotary, o1_rope_turns) against complex arithmetic in 64 bits.

Bounds, from the arithmetic: a frequency's fraction of a turn is rounded to 2^-65, its product with the position is exact; the rest of an angle, below pi / 4, has fp32's rounding
twice (2^-23 of it), sine and cosine that, 2.5e-8 of the polynomials' rest and three roundings: together below 2^-22.  With two products of which one is rounded and a sum, a
result is within (|a| + |b|) * factor * 2^-21 of the 64-bit one, then rounded to its type once."""
import ctypes as C
import math
from decimal import Decimal, getcontext

import pytest
import torch

gpu = pytest.mark.gpu
getcontext().prec = 60
PI = Decimal("3.14159265358979323846264338327950288419716939937510582097494")
THETA = 5000000.0


def gen(seed):
    return torch.Generator().manual_seed(seed)


def frequencies(rot, theta=THETA, scaling=None):
    """By the definition, in decimals of sixty places."""
    s = scaling or {"kind": "none"}
    by = Decimal(s.get("factor", 1.0))
    base = Decimal(theta)
    if s["kind"] == "ntk":
        base *= by ** (Decimal(rot) / Decimal(max(rot - 2, 1)))
    f = [base ** (-Decimal(2 * i) / rot) for i in range(rot // 2)]
    if s["kind"] == "linear":
        f = [x / by for x in f]
    if s["kind"] == "yarn":
        def pair_at(t):
            return rot * math.log(s["original"] / (t * 2 * math.pi)) / (2 * math.log(theta))
        low, high = max(math.floor(pair_at(s.get("fast", 32.0))), 0), min(math.ceil(pair_at(s.get("slow", 1.0))), rot - 1)
        for i in range(rot // 2):
            ramp = Decimal(min(max((i - low) / max(high - low, 0.001), 0.0), 1.0))
            f[i] = f[i] / by * ramp + f[i] * (1 - ramp)
    if s["kind"] == "factors":
        f = [x / Decimal(d) for x, d in zip(f, s["factors"])]
    return f


SCALINGS = [None, {"kind": "linear", "factor": 8.0}, {"kind": "ntk", "factor": 4.0}, {"kind": "yarn", "factor": 16.0, "original": 4096.0},
            {"kind": "yarn", "factor": 2.0, "original": 300.0, "fast": 4.0, "slow": 0.5, "attention": 1.25}]


def turns_of(pkg, rot, theta=THETA, scaling=None):
    s = scaling or {"kind": "none"}
    factors = s.get("factors")
    c = pkg.RopeScalingC({"none": 0, "linear": 1, "ntk": 2, "yarn": 3, "factors": 4}[s["kind"]], s.get("factor", 1.0), s.get("original", 0.0), s.get("fast", 32.0),
                         s.get("slow", 1.0), s.get("attention", 0.0), (C.c_double * len(factors))(*factors) if factors else None)
    turns, factor = (C.c_uint64 * max(rot // 2, 1))(), C.c_float()
    rc = pkg.lib.o1_rope_turns(theta, rot, C.byref(c), turns, C.byref(factor))
    return rc, list(turns), factor.value


@pytest.mark.parametrize("rot,theta", [(128, THETA), (64, 10000.0), (2, 500.0), (72, 1.5), (4, 10000.0)])
@pytest.mark.parametrize("scaling", SCALINGS)
def test_frequencies_as_turns(pkg, rot, theta, scaling):
    """Within 2^-61 of a frequency (long double's powers) and 2^-64 turns; the factor of results."""
    if scaling and scaling["kind"] == "yarn" and theta < 2:
        theta = 10000.0
    rc, turns, factor = turns_of(pkg, rot, theta, scaling)
    assert rc == 0
    for t, f in zip(turns, frequencies(rot, theta, scaling)):
        want = f / (2 * PI)
        off = (Decimal(t) / 2 ** 64 - want) % 1
        assert min(off, 1 - off) <= want * Decimal(2.0 ** -58) + Decimal(2.0 ** -64), (t, f)
    want = 1.0 if not scaling else scaling.get("attention", 0.1 * math.log(scaling["factor"]) + 1.0 if scaling["kind"] == "yarn" else 1.0)
    assert abs(factor - want) <= 1e-7 * want


def test_one_factor_for_each_pair(pkg):
    s = {"kind": "factors", "factors": [1.0 + 0.5 * i for i in range(16)]}
    rc, turns, factor = turns_of(pkg, 32, 10000.0, s)
    assert rc == 0 and factor == 1.0
    for t, f in zip(turns, frequencies(32, 10000.0, s)):
        assert abs(Decimal(t) / 2 ** 64 - f / (2 * PI)) <= Decimal(2.0 ** -60)


def test_entry_points_refuse_before_they_touch_the_gpu(pkg):
    lib, one = pkg.lib, C.c_void_p(4096)
    for rot, theta, s in ((0, THETA, None), (3, THETA, None), (-2, THETA, None), (1 << 20, THETA, None), (8, 1.0, None), (8, math.nan, None), (8, THETA, {"kind": "linear", "factor": 0.5}),
                          (8, THETA, {"kind": "ntk", "factor": math.nan}), (8, THETA, {"kind": "yarn", "factor": 2.0, "original": 0.0}),
                          (8, THETA, {"kind": "yarn", "factor": 2.0, "original": 100.0, "fast": 1.0, "slow": 2.0}), (8, THETA, {"kind": "factors", "factors": [1.0, 0.0, 1.0, 1.0]})):
        assert turns_of(pkg, rot, theta, s)[0] == 9, (rot, theta, s)
        assert b"rope_turns" in lib.hd_cuda_last_error()
    assert lib.o1_rope_turns(THETA, 8, None, None, None) == 6

    def call(pos=one, wide=0, x=one, ldx=256, y=one, ldy=256, heads=2, x2=None, ld2=0, y2=None, heads2=0, rows=3, type_=0, **change):
        r = pkg.RopeC(**{**dict(turns=4096, factor=1.0, head_dim=128, rot_dim=128, layout=0), **change})
        return lib.o1_rotary(C.byref(r), pos, wide, x, ldx, y, ldy, heads, x2, ld2, y2, ld2, heads2, rows, type_, 0)

    for want, args in ((6, dict(pos=None)), (6, dict(x=None)), (6, dict(y=None)), (6, dict(heads2=1, ld2=128)), (6, dict(turns=None)), (9, dict(rot_dim=127)), (9, dict(rot_dim=130)),
                       (9, dict(rot_dim=0)), (9, dict(head_dim=0)), (9, dict(head_dim=8192, rot_dim=64)), (9, dict(layout=2)), (9, dict(type_=2)), (9, dict(rows=-1)), (9, dict(heads=-1)),
                       (9, dict(ldx=255)), (9, dict(ldy=0)), (9, dict(heads2=2, x2=one, y2=one, ld2=255)), (9, dict(heads=70000, ldx=70000 * 128, ldy=70000 * 128)),
                       (9, dict(x=C.c_void_p(4097))), (9, dict(x=C.c_void_p(4098), type_=1)), (9, dict(pos=C.c_void_p(4098))), (9, dict(pos=C.c_void_p(4100), wide=1))):
        assert call(**args) == want, args
        assert b"rotary" in lib.hd_cuda_last_error(), args
    assert lib.o1_rotary(None, one, 0, one, 256, one, 256, 2, None, 0, None, 0, 0, 1, 0, 0) == 6
    assert call(rows=0) == 0 and call(heads=0) == 0
    lib.hd_cuda_clear_error()


def reference(rope, x, positions, inverse=False):
    """The 64-bit result and the bound, with the angles that the kept turns stand for."""
    half, rot = rope.rot_dim // 2, rope.rot_dim
    turns = [t % 2 ** 64 for t in rope.turns.tolist()]
    angle = torch.tensor([[(p * t % 2 ** 64) / 2 ** 64 for t in turns] for p in positions.tolist()], dtype=torch.float64).view(-1, half) * (2 * math.pi)
    first = torch.arange(half) * (1 if rope.layout == "half" else 2)
    second = first + (half if rope.layout == "half" else 1)
    x = x.cpu().double()
    z = torch.complex(x[..., first], x[..., second]) * torch.polar(torch.full_like(angle, rope.factor), -angle if inverse else angle)[:, None]
    y, tol = x.clone(), torch.zeros_like(x)
    y[..., first], y[..., second] = z.real, z.imag
    tol[..., first] = tol[..., second] = (x[..., first].abs() + x[..., second].abs()) * rope.factor * 2.0 ** -21
    return y, tol


def check(rope, x, got, positions, inverse=False):
    assert got.dtype == x.dtype and got.shape == x.shape
    ref, tol = reference(rope, x, positions, inverse)
    got = got.cpu()
    assert ((got.double() >= (ref - tol).to(x.dtype).double()) & (got.double() <= (ref + tol).to(x.dtype).double())).all(), ((got.double() - ref).abs() / (tol + 1e-300)).max()
    assert torch.equal(got[..., rope.rot_dim:], x.cpu()[..., rope.rot_dim:])


def normal(shape, g, dtype):
    return torch.randn(shape, generator=g).to(dtype)


@gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("layout", ["half", "interleaved"])
@pytest.mark.parametrize("head,rot", [(128, 128), (128, 64), (64, 64), (72, 72), (96, 96), (96, 2), (256, 256), (2, 2), (3, 2), (80, 34), (128, 112), (136, 16), (4096, 64)])
def test_layouts_and_parts_of_a_head(pkg, dev, dtype, layout, head, rot):
    rope = pkg.Rotary(head, rot, THETA, layout, device=dev)
    for rows, heads, kv in ((1, 1, 1), (5, 4, 1), (33, 3, 2)):
        q, k = normal((rows, heads, head), gen(rows), dtype).to(dev), normal((rows, kv, head), gen(9), dtype).to(dev)
        pos = torch.arange(rows, dtype=torch.int32) * 37
        got_q, got_k = rope((q, k), pos.to(dev))
        check(rope, q, got_q, pos)
        check(rope, k, got_k, pos)
        assert torch.equal(rope(q, pos.to(dev)), got_q) and torch.equal(rope(q, pos.long().to(dev)), got_q)


@gpu
@pytest.mark.parametrize("scaling", SCALINGS)
@pytest.mark.parametrize("layout", ["half", "interleaved"])
def test_far_and_negative_positions(pkg, dev, scaling, layout):
    rope = pkg.Rotary(64, 64, 10000.0, layout, scaling, device=dev)
    pos = torch.tensor([0, 1, -1, 4095, 16640, 10 ** 6, -10 ** 6, 2 ** 31 - 1, -2 ** 31, 2 ** 40 + 12345, -2 ** 62, 2 ** 63 - 1])
    x = normal((len(pos), 3, 64), gen(1), torch.float32).to(dev)
    check(rope, x, rope(x, pos.to(dev)), pos)
    near = pos.clamp(-2 ** 31, 2 ** 31 - 1)
    assert torch.equal(rope(x, near.int().to(dev)), rope(x, near.to(dev)))


@gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("rows,heads,kv", [(1, 32, 8), (24, 32, 8), (1000, 32, 8), (3001, 7, 1), (700, 128, 128)])
def test_few_and_many_rows(pkg, dev, dtype, rows, heads, kv):
    """Heads to a thread and rows to a block of each size; a few rows are looked at."""
    rope = pkg.Rotary(128, device=dev)
    q, k = normal((rows, heads, 128), gen(rows), dtype).to(dev), normal((rows, kv, 128), gen(9), dtype).to(dev)
    pos = (torch.arange(rows, dtype=torch.int32) * 7919) % 16640
    got = rope((q, k), pos.to(dev))
    some = torch.unique(torch.tensor([0, 1, rows // 2, rows - 2, rows - 1]).clamp(0, rows - 1))
    for x, y in zip((q, k), got):
        check(rope, x[some.to(dev)], y[some.to(dev)], pos[some])
        alone = rope(x, pos.to(dev))
        assert torch.equal(alone, y)
    assert torch.equal(torch.cat([rope(q[i:i + 1], pos[i:i + 1].to(dev)) for i in some.tolist()]), got[0][some.to(dev)])


@gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("off,pad", [(0, 0), (0, 16), (1, 0), (4, 4), (3, 5)])
def test_rows_inside_wider_ones_and_in_place(pkg, dev, dtype, off, pad):
    rows, heads, kv, head = 29, 4, 2, 96
    rope = pkg.Rotary(head, 64, layout="half", device=dev)
    pitch = (heads + 2 * kv) * head + pad
    wide = torch.randn(rows * pitch + off, generator=gen(1)).to(dtype).to(dev)
    before = wide.clone()
    w = wide[off:].view(rows, pitch)
    q, k = w[:, :heads * head].unflatten(1, (heads, head)), w[:, heads * head:(heads + kv) * head].unflatten(1, (kv, head))
    pos = torch.arange(rows, dtype=torch.int32, device=dev) + 1000
    want = rope((q.contiguous(), k.contiguous()), pos)
    got = rope((q, k), pos)
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1]) and torch.equal(wide, before)
    back = rope((q, k), pos, out=(q, k))
    assert back[0].data_ptr() == q.data_ptr() and torch.equal(q, want[0]) and torch.equal(k, want[1])
    assert torch.equal(w[:, (heads + kv) * head:], before[off:].view(rows, pitch)[:, (heads + kv) * head:]) and torch.equal(wide[:off], before[:off])


@gpu
@pytest.mark.parametrize("layout", ["half", "interleaved"])
def test_turned_back_is_the_gradient(pkg, dev, layout):
    """The adjoint by the formula, and against differences of a scalar function of the results."""
    rope = pkg.Rotary(48, 32, 10000.0, layout, {"kind": "yarn", "factor": 4.0, "original": 128.0}, device=dev)
    pos = torch.arange(11, dtype=torch.int32) * 91
    x, g = (normal((11, 3, 48), gen(i), torch.float32).to(dev) for i in (1, 2))
    back = rope(g, pos.to(dev), inverse=True)
    check(rope, g, back, pos, inverse=True)
    d, step = normal(x.shape, gen(3), torch.float32).to(dev), 2.0 ** -4
    ahead, behind = ((g.double() * rope(x + s * step * d, pos.to(dev)).double()).sum() for s in (1, -1))
    # a linear function: the difference is exact but for roundings, of 2^-22 of some 1600 terms of about 2 each
    assert abs(float((ahead - behind) / (2 * step) - (back.double() * d.double()).sum())) < 2.0 ** -20 / step * 4 * x.numel()
    y = rope(rope(x, pos.to(dev)), pos.to(dev), inverse=True)[..., :32].double() / rope.factor ** 2
    assert (y - x[..., :32].double()).abs().max() < 2.0 ** -18 * float(x.abs().max())


@gpu
def test_not_finite_values_stay_in_their_pair(pkg, dev):
    rope = pkg.Rotary(128, 64, device=dev)
    x = normal((3, 2, 128), gen(1), torch.bfloat16)
    x[1, 0, 5], x[2, 1, 100] = math.nan, math.inf
    y = rope(x.to(dev), torch.tensor([1, 2, 3], dtype=torch.int32, device=dev)).cpu()
    bad = ~torch.isfinite(y)
    assert bad.sum() == 3 and bad[1, 0, 5] and bad[1, 0, 37] and y[2, 1, 100] == math.inf


@gpu
def test_streams_and_graphs(pkg, dev):
    rope = pkg.Rotary(device=dev)
    x, pos = normal((9, 4, 128), gen(1), torch.bfloat16).to(dev), torch.arange(9, dtype=torch.int32, device=dev)
    want, later = rope(x, pos), rope(x, pos + 500)
    y, s = torch.empty_like(x), torch.cuda.Stream()
    torch.cuda.synchronize()
    try:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=s):
            pkg.use_torch_stream()
            rope(x, pos, out=y)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(y, want)
        pos += 500
        graph.replay()
        torch.cuda.synchronize()
    finally:
        pkg.use_torch_stream()
    assert torch.equal(y, later)


@gpu
def test_arguments_that_do_not_fit(pkg, dev):
    E = pkg.O1Error
    for args in ((128, 130), (128, 63), (128, 0), (8192, 64)):
        with pytest.raises(E, match="rot_dim"):
            pkg.Rotary(*args, device=dev)
    with pytest.raises(E, match="layout"):
        pkg.Rotary(layout="both", device=dev)
    for s in ({"kind": "other"}, {"factor": 2.0}, {"kind": "linear", "by": 2.0}, {"kind": "factors", "factors": [1.0]}, {"kind": "linear", "factor": 2.0, "factors": [1.0] * 64}):
        with pytest.raises(E, match="Rotary"):
            pkg.Rotary(scaling=s, device=dev)
    with pytest.raises(E, match="rope_turns"):
        pkg.Rotary(scaling={"kind": "linear", "factor": 0.0}, device=dev)
    rope = pkg.Rotary(128, device=dev)
    x, pos = torch.zeros(3, 2, 128, dtype=torch.bfloat16, device=dev), torch.zeros(3, dtype=torch.int32, device=dev)
    for bad in (x[0], x[..., :64], x.half(), x.cpu(), x[:2], x.transpose(0, 1).contiguous().transpose(0, 1)):
        with pytest.raises(E, match="Rotary"):
            rope(bad, pos)
    for bad in (pos.float(), pos[:2], pos.cpu(), pos[None], pos.repeat(2)[::2]):
        with pytest.raises(E, match="Rotary"):
            rope(x, bad)
    with pytest.raises(E, match="Rotary"):
        rope((x, x.float()), pos)
    with pytest.raises(E, match="Rotary"):
        rope((x, x, x), pos)
    with pytest.raises(E, match="Rotary"):
        rope(x, pos, out=x[:, :1])
    assert rope(x[:0], pos[:0]).shape == (0, 2, 128) and rope(x[:, :0], pos).shape == (3, 0, 128)
    pkg.check_cuda_errbuf("after refusals")


@gpu
@pytest.mark.parametrize("theta,scaling", [(THETA, {"kind": "linear", "factor": 8.0}), (THETA, {"kind": "yarn", "factor": 32.0, "original": 16640.0}), (1.0e9, None), (10000.0, None)])
@pytest.mark.parametrize("layout", ["half", "interleaved"])
def test_sines_keep_their_bits(pkg, dev, theta, scaling, layout):
    """Pairs (1, 0) and (0, 1) in fp32 give sines and cosines themselves, small ones too: within 2^-21 of their own size (an angle's rounding to fp32, a constant's, a product's, a sum's, two of the
    polynomial's, one with the factor: seven of 2^-24, and the polynomials' rest, 2.5e-8)."""
    rot = 128
    rope = pkg.Rotary(rot, rot, theta, layout, scaling, dev)
    positions = [0, 1, 2, 3, 5, 17, 100, 1000, 16640, 999983, -1, -3, 2 ** 31 - 1, -2 ** 31, 2 ** 45 + 1, -2 ** 62 + 3]
    first = torch.arange(rot // 2) * (1 if layout == "half" else 2)
    second = first + (rot // 2 if layout == "half" else 1)
    x = torch.zeros(len(positions), 2, rot)
    x[:, 0, first], x[:, 1, second] = 1.0, 1.0
    got = rope(x.to(dev), torch.tensor(positions, device=dev)).cpu().double()
    sin, cos = (torch.zeros(len(positions), rot // 2, dtype=torch.float64) for _ in range(2))
    for i, p in enumerate(positions):
        for j, t in enumerate(rope.turns.tolist()):
            t = p * (t % 2 ** 64) % 2 ** 64
            quarter = (t + 2 ** 61) // 2 ** 62
            a = (t - quarter * 2 ** 62) * (math.pi / 2 ** 63)
            s, c = ((math.sin(a), math.cos(a)), (math.cos(a), -math.sin(a)), (-math.sin(a), -math.cos(a)), (-math.cos(a), math.sin(a)))[quarter % 4]
            sin[i, j], cos[i, j] = s * rope.factor, c * rope.factor
    for g, want in ((got[:, 0, first], cos), (got[:, 0, second], sin), (got[:, 1, first], -sin), (got[:, 1, second], cos)):
        assert ((g - want).abs() <= 2.0 ** -21 * want.abs()).all(), ((g - want).abs() / want.abs().clamp_min(1e-300)).max()


# (columns of a buffer of 1024-value rows: from, heads, first row) of x, y, x2, y2, heads of 128; rows 4
MEMORY = [(False, [(0, 2, 0), (128, 2, 0)]), (False, [(0, 2, 0), (0, 2, 1)]), (False, [(0, 2, 1), (0, 2, 0)]), (False, [(0, 2, 0), (1024 - 128, 2, 0)]), (False, [(1024 - 128, 2, 0), (0, 2, 1)]),
          (False, [(0, 2, 0), (0, 2, 3)]), (False, [(0, 2, 0), (0, 2, 0), (128, 1, 0), (512, 1, 0)]), (False, [(0, 2, 0), (512, 2, 0), (256, 1, 0), (0, 1, 0)]),
          (False, [(0, 2, 0), (512, 2, 0), (256, 1, 0), (640, 1, 0)]), (False, [(0, 2, 0), (0, 2, 0), (0, 2, 0), (0, 2, 0)]), (False, [(0, 2, 0), (512, 2, 0), (512, 2, 0), (0, 2, 0)]),
          (True, [(0, 2, 0), (0, 2, 0)]), (True, [(0, 2, 0), (256, 2, 0)]), (True, [(256, 2, 0), (0, 2, 0)]), (True, [(0, 2, 0), (0, 2, 4)]), (True, [(0, 2, 4), (0, 2, 0)]),
          (True, [(0, 2, 0), (0, 2, 0), (256, 1, 0), (256, 1, 0)]), (True, [(0, 2, 0), (256, 2, 0), (0, 2, 0), (512, 2, 0)]), (True, [(0, 2, 0), (256, 2, 2), (512, 1, 1), (640, 1, 3)]),
          (True, [(768, 2, 0), (0, 2, 1)])]


@pytest.mark.parametrize("case", [c for ok, c in MEMORY if not ok])
def test_results_over_other_rows_are_refused(pkg, case):
    at = [C.c_void_p(4096 + 2 * (row * 1024 + column)) for column, _, row in case] + [None] * (4 - len(case))
    heads = [h for _, h, _ in case] + [0, 0]
    r = pkg.RopeC(turns=4096, factor=1.0, head_dim=128, rot_dim=128, layout=0)
    assert pkg.lib.o1_rotary(C.byref(r), C.c_void_p(4096), 0, at[0], 1024, at[1], 1024, heads[0], at[2], 1024, at[3], 1024, heads[2], 4, 0, 0) == 9
    assert b"share memory" in pkg.lib.hd_cuda_last_error()
    pkg.lib.hd_cuda_clear_error()


def test_results_over_other_rows_of_another_pitch_are_refused(pkg):
    """Rows 1024 apart into rows of other pitches, against every address of both."""
    r = pkg.RopeC(turns=4096, factor=1.0, head_dim=16, rot_dim=16, layout=0)
    refused = 0
    for ldy in (16, 24, 40, 56, 64, 200):
        for off in range(-200, 200, 8):
            x = {(i * 48 + j) for i in range(4) for j in range(16)}
            y = {(off + i * ldy + j) for i in range(4) for j in range(16)}
            if not x & y:
                continue           # (nothing that would be launched)
            refused += 1
            assert pkg.lib.o1_rotary(C.byref(r), C.c_void_p(4096), 0, C.c_void_p(8192), 48, C.c_void_p(8192 + 2 * off), ldy, 1, None, 0, None, 0, 0, 4, 0, 0) == 9, (ldy, off)
    assert refused > 60
    pkg.lib.hd_cuda_clear_error()


@gpu
@pytest.mark.parametrize("case", [c for ok, c in MEMORY if ok])
def test_results_beside_other_rows(pkg, dev, case):
    rope = pkg.Rotary(128, device=dev)
    wide = torch.randn(9, 1024, generator=gen(1)).bfloat16().to(dev)
    pos = torch.arange(4, dtype=torch.int32, device=dev) + 5
    views = [wide[row:row + 4, column:column + h * 128].unflatten(1, (h, 128)) if column + h * 128 <= 1024 else None for column, h, row in case]
    want = [rope(x.clone(), pos) for x in views[::2]]
    if len(case) == 2:
        rope(views[0], pos, out=views[1])
    else:
        rope((views[0], views[2]), pos, out=(views[1], views[3]))
    for y, w in zip(views[1::2], want):
        assert torch.equal(y, w)


@gpu
def test_results_between_rows_of_another_pitch(pkg, dev):
    """Every pitch and offset that shares nothing with the rows, in one buffer."""
    rope = pkg.Rotary(16, device=dev)
    pos = torch.arange(4, dtype=torch.int32, device=dev) + 5
    done = 0
    for ldy in (16, 24, 40, 48, 56, 64, 200):
        for off in range(-200, 200, 8):
            if {(i * 48 + j) for i in range(4) for j in range(16)} & {(off + i * ldy + j) for i in range(4) for j in range(16)}:
                continue
            done += 1
            buf = torch.randn(1200, generator=gen(done)).bfloat16().to(dev)
            x, y = buf[200:].as_strided((4, 1, 16), (48, 16, 1), 200), buf.as_strided((4, 1, 16), (ldy, 16, 1), 200 + off)
            want = rope(x.clone(), pos)
            assert torch.equal(rope(x, pos, out=y), want)
    assert done > 100


# ------------------------------------------------------------------ gradients
@gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("layout", ["half", "interleaved"])
@pytest.mark.parametrize("inverse", [False, True])
def test_rows_that_need_a_gradient(pkg, dev, dtype, layout, inverse):
    """Results' gradients turned back, by the formula in 64 bits: of one tensor, of both of a pair, of one of a pair, of slices of wider rows, with gradients of any layout."""
    rope = pkg.Rotary(96, 64, 10000.0, layout, {"kind": "yarn", "factor": 4.0, "original": 128.0}, dev)
    pos = torch.arange(13, dtype=torch.int32) * 91
    at = pos.to(dev)
    q, k, gq, gk = (normal((13, h, 96), gen(i), dtype).to(dev) for i, h in enumerate((4, 2, 4, 2)))
    plain = rope((q, k), at, inverse)
    q.requires_grad_(), k.requires_grad_()
    y = rope(q, at, inverse)
    assert torch.equal(y, plain[0]) and y.requires_grad
    y.backward(gq)
    check(rope, gq, q.grad, pos, inverse=not inverse)
    for need in ((True, True), (True, False), (False, True)):
        x = [t.detach().clone().requires_grad_(n) for t, n in zip((q, k), need)]
        ys = rope(tuple(x), at, inverse)
        assert all(torch.equal(a, b) for a, b in zip(ys, plain))
        (ys[0].float() * gq.float()).sum().add((ys[1].float() * gk.float()).sum()).backward()
        for t, g, n in zip(x, (gq, gk), need):
            assert (t.grad is not None) == n
            if n:
                check(rope, g, t.grad, pos, inverse=not inverse)
    wide = normal((13, 6 * 96), gen(9), dtype).to(dev).requires_grad_()
    a, b = rope((wide[:, :4 * 96].unflatten(1, (4, 96)), wide[:, 4 * 96:].unflatten(1, (2, 96))), at, inverse)
    torch.autograd.backward((a, b), (gq.transpose(0, 1).contiguous().transpose(0, 1), gk))
    check(rope, torch.cat([gq, gk], 1), wide.grad.unflatten(1, (6, 96)), pos, inverse=not inverse)
    one = q.detach().clone().requires_grad_()
    rope(one, at, inverse).sum().backward()            # (a gradient of one value for all)
    check(rope, torch.ones_like(one), one.grad, pos, inverse=not inverse)
    used = [t.detach().clone().requires_grad_() for t in (q, k)]
    rope(tuple(used), at, inverse)[1].backward(gk)      # (the other one's result is not used)
    check(rope, gk, used[1].grad, pos, inverse=not inverse)
    assert used[0].grad is None or not used[0].grad.any()


@gpu
def test_a_gradient_against_differences(pkg, dev):
    """Of a function that is not linear: sum of g * y^2 / 2, whose second derivatives are known too (the gradient of a gradient)."""
    rope = pkg.Rotary(32, 24, 10000.0, "interleaved", device=dev)
    at = torch.arange(7, dtype=torch.int32, device=dev) * 5
    x, g, d = (normal((7, 2, 32), gen(i), torch.float32).to(dev) for i in (1, 2, 3))
    x.requires_grad_()

    def f(t):
        return (g.double() * rope(t, at).double().square()).sum() / 2

    grad, = torch.autograd.grad(f(x), x, create_graph=True)
    step = 2.0 ** -4
    with torch.no_grad():
        along = (f(x + step * d) - f(x - step * d)) / (2 * step)
    # quadratic: the difference is exact but for roundings, 2^-20 of some 450 terms of about 4 each, in y and in the gradient
    assert abs(float((grad.detach().double() * d.double()).sum() - along)) < 2.0 ** -20 / step * 4 * x.numel()
    second, = torch.autograd.grad((grad * d).sum(), x)
    with torch.no_grad():
        want = rope(g * rope(d, at), at, inverse=True)
    assert (second - want).abs().max() < 2.0 ** -18 * float(want.abs().max())


@gpu
def test_no_gradient_where_none_is_wanted(pkg, dev):
    rope = pkg.Rotary(64, device=dev)
    at = torch.arange(3, dtype=torch.int32, device=dev)
    x = normal((3, 2, 64), gen(1), torch.float32).to(dev).requires_grad_()
    want = rope(x.detach(), at)
    with torch.no_grad():
        assert not rope(x, at).requires_grad and torch.equal(rope(x, at, out=torch.empty_like(want)), want)
    with torch.inference_mode():
        assert torch.equal(rope((x, x), at)[1], want)
    for call in (lambda: rope(x, at, out=torch.empty_like(want)), lambda: rope(x * 1.0, at, out=x), lambda: rope(want, at, out=torch.empty_like(want).requires_grad_()),
                 lambda: rope((want, x), at, out=(torch.empty_like(want), torch.empty_like(want)))):
        with pytest.raises(pkg.O1Error, match="gradient"):
            call()


@gpu
def test_gradients_on_streams_and_in_graphs(pkg, dev):
    """Backward on the stream that autograd takes, wherever the library's is by then; forward and backward as one graph, replayed with other rows, gradients and positions."""
    rope = pkg.Rotary(64, device=dev)
    pos = torch.arange(300, dtype=torch.int32, device=dev)
    x, g = (normal((300, 8, 64), gen(i), torch.float32).to(dev) for i in (1, 2))
    want, s = rope(g, pos, inverse=True), torch.cuda.Stream()
    torch.cuda.synchronize()
    try:
        leaf = x.clone().requires_grad_()
        torch.cuda.synchronize()
        with torch.cuda.stream(s):
            pkg.use_torch_stream()
            y = rope(leaf, pos)
        pkg.use_torch_stream()
        torch.cuda.synchronize()
        back, = torch.autograd.grad(y, leaf, g)
        torch.cuda.synchronize()
        assert torch.equal(back, want) and pkg.lib.o1_get_stream() in (None, torch.cuda.current_stream().cuda_stream)
        del y, leaf
        static = x.clone().requires_grad_()
        graph = torch.cuda.CUDAGraph()
        torch.cuda.synchronize()
        with torch.cuda.graph(graph, stream=s):
            pkg.use_torch_stream()
            y = rope(static, pos)
            back, = torch.autograd.grad(y, static, g)
    finally:
        pkg.use_torch_stream()
    for i in range(3):
        with torch.no_grad():
            static.copy_(x * (i + 1)), g.mul_(-2.0), pos.add_(11)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(y, rope(static.detach(), pos)) and torch.equal(back, rope(g, pos, inverse=True))


@gpu
def test_scalings_that_would_be_passed_over_are_refused(pkg, dev):
    """A factor left out was 1, and a factor of results that is not positive was the method's own; an infinite one gave infinities."""
    for s in ({"kind": "linear"}, {"kind": "ntk"}, {"kind": "yarn", "original": 4096.0}, *({"kind": "yarn", "factor": 4.0, "original": 4096.0, "attention": a} for a in (0.0, -1.0, math.nan, math.inf)),
              {"kind": "none", "attention": 0}):
        with pytest.raises(pkg.O1Error, match="Rotary"):
            pkg.Rotary(64, scaling=s, device=dev)
    assert pkg.Rotary(64, scaling={"kind": "none", "attention": 1.5}, device=dev).factor == 1.5
    assert pkg.Rotary(64, scaling={"kind": "factors", "factors": [2.0] * 32}, device=dev).factor == 1.0
