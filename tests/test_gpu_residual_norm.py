"""residual_norm (y = x + alpha * gate * u, h = norm(y)) against 64-bit arithmetic.

Tolerances: y and h are rounded once, so they lie between the ends, as rounded, of what a handful of fp32 operations before that
may be off by: 2^-20 of the terms they sum."""
import ctypes as C
import math

import pytest
import torch

from test_gpu_kvcache import between

gpu = pytest.mark.gpu


def normal(shape, seed, std=1.0, mean=0.0):
    return (torch.randn(shape, generator=torch.Generator().manual_seed(seed)) * std + mean).to(torch.bfloat16)


def reference(x, b, pre, post, gate, scale, shift, alpha, eps):
    def norm(a, w):
        return a / torch.sqrt((a * a).mean(-1, keepdim=True) + eps) * w.double()

    def each(v):
        v = v.double().reshape(-1, x.shape[1])
        return v.repeat_interleave(x.shape[0] // v.shape[0], 0)

    u = b.double() if post is None else norm(b.double(), post)
    u = alpha * (u if gate is None else u * each(gate))
    y = x.double() + u
    tol_y = (x.double().abs() + u.abs()) * 2.0 ** -20
    if pre is None:
        return y, None, tol_y, None
    h = norm(y, pre)
    # an error of y's terms is one of h's, times inv * pre
    slip = (x.double().abs() + u.abs()) * 2.0 ** -20 * (h / torch.where(y == 0, 1.0, y)).abs() + h.abs() * 2.0 ** -19
    if scale is not None:
        s = 1 + each(scale)
        slip = slip * s.abs() + ((h * s).abs() + each(shift).abs()) * 2.0 ** -20
        h = h * s + each(shift)
    return y, h, tol_y, slip


CASES = [(1, 4096, 0, 0, 0), (3, 4096, 1, 1, 1), (592, 4096, 1, 2, 1), (7, 8, 1, 1, 1), (5, 1, 1, 1, 1), (33, 1152, 1, 1, 0), (130, 1024, 0, 2, 1), (9, 1000, 1, 3, 1),
         (12, 1001, 1, 3, 1), (4, 4104, 1, 2, 0), (6, 8192, 1, 1, 1), (3, 8200, 1, 1, 1), (2, 12288, 0, 0, 1), (257, 64, 0, 1, 1), (4100, 72, 1, 0, 0), (3, 20000, 1, 3, 1)]


@gpu
@pytest.mark.parametrize("rows,cols,post,groups,mod", CASES)
@pytest.mark.parametrize("layout", ["plain", "pitched", "odd"])
def test_against_64_bits(pkg, dev, rows, cols, post, groups, mod, layout):
    pitch, off = {"plain": (cols, 0), "pitched": (cols + 16, 0), "odd": (cols + 3, 1)}[layout]
    alpha = 0.37
    x, b = normal((rows, cols), 1, 2.0), normal((rows, cols), 2, 0.7)
    pre, pw = normal((cols,), 3, 0.2, 1.0), normal((cols,), 4, 0.2, 1.0) if post else None
    n = max(groups, 1)
    gate = normal((n, cols), 5, 0.6) if groups else None
    scale, shift = (normal((n, cols), 6, 0.3), normal((n, cols), 7, 0.3)) if mod else (None, None)

    def place(t):
        buf = torch.full((rows * pitch + off,), 9.0, dtype=torch.bfloat16, device=dev)
        view = buf[off:].view(rows, pitch)[:, :cols]
        if t is not None:
            view.copy_(t)
        return buf, view

    d = lambda t: None if t is None else t.to(dev)  # noqa: E731
    (_, xd), (_, bd), (ybuf, yd), (hbuf, hd) = place(x), place(b), place(None), place(None)
    y, h = pkg.residual_norm(xd, bd, d(pre), post_w=d(pw), gate=d(gate), scale=d(scale), shift=d(shift), alpha=alpha, eps=1e-6, y=yd, h=hd)
    ry, rh, ty, th = reference(x, b, pre, pw, gate, scale, shift, alpha, 1e-6)
    for name, got, ref, tol in (("y", y, ry, ty), ("h", h, rh, th)):
        between(got, ref, tol, name)
    for buf in (ybuf, hbuf):
        if pitch > cols:
            assert (buf[off:].view(rows, pitch)[:, cols:] == 9.0).all()
        assert (buf[:off] == 9.0).all()
    y2, h2 = pkg.residual_norm(xd, bd, d(pre), post_w=d(pw), gate=d(gate), scale=d(scale), shift=d(shift), alpha=alpha, eps=1e-6)
    assert torch.equal(y, y2) and torch.equal(h, h2)
    # in place, and without the second norm
    y3, h3 = pkg.residual_norm(xd, bd, None, post_w=d(pw), gate=d(gate), alpha=alpha, y=xd)
    assert h3 is None and torch.equal(xd, y2) and y3.data_ptr() == xd.data_ptr()


@gpu
@pytest.mark.parametrize("cols", [4096, 1001])
def test_rows_that_are_not_ordinary(pkg, dev, cols):
    """Rows of zeros, of 2^-120 and of 2^60; a NaN stays in its row."""
    x, b = normal((5, cols), 1), normal((5, cols), 2)
    x[0], b[0] = 0, 0
    x[1], b[1] = x[1] * 2.0 ** -120, b[1] * 2.0 ** -120
    x[2], b[2] = x[2] * 2.0 ** 60, b[2] * 2.0 ** 60
    x[3, 3] = math.nan
    pre, post = normal((cols,), 3, 0.1, 1.0), normal((cols,), 4, 0.1, 1.0)
    y, h = pkg.residual_norm(x.to(dev), b.to(dev), pre.to(dev), post_w=post.to(dev))
    ry, rh, ty, th = reference(x, b, pre, post, None, None, None, 1.0, 1e-6)
    good = [0, 1, 2, 4]
    assert (y[0] == 0).all() and (h[0] == 0).all()
    between(y[good], ry[good], (ty + 1e-37)[good], "y")
    between(h[good], rh[good], (th + 1e-37)[good], "h")
    assert torch.isnan(h[3]).all() and torch.isnan(y[3]).sum() == 1


@gpu
def test_a_block_s_own_two_calls(pkg, dev):
    """Beside hd_residual_add and hd_rmsnorm: y is the same, h differs by the rounding of y that those have between them."""
    x, b, w = normal((70, 4096), 1).to(dev), normal((70, 4096), 2).to(dev), normal((4096,), 3, 0.1, 1.0).to(dev)
    y0, h0 = torch.empty_like(x), torch.empty_like(x)
    pkg.lib.hd_residual_add(pkg.ptr(x), pkg.ptr(b), pkg.ptr(y0), x.numel())
    pkg.lib.hd_rmsnorm(pkg.ptr(y0), pkg.ptr(w), pkg.ptr(h0), 70, 4096, 1e-6)
    y, h = pkg.residual_norm(x, b, w)
    assert torch.equal(y, y0)
    assert ((h.float() - h0.float()).abs() <= h0.float().abs() * 2.0 ** -7 + 1e-3).all()


@gpu
def test_arguments_that_do_not_fit(pkg, dev):
    E, x, w = pkg.O1Error, normal((4, 64), 1).to(dev), normal((64,), 2).to(dev)
    m3, m2 = normal((3, 64), 2).to(dev), normal((2, 64), 2).to(dev)
    for args, kw in (((x.float(), x, w), {}), ((x, x[:2], w), {}), ((x, x, w[:32]), {}), ((x, x, w.float()), {}), ((x, x, w), dict(gate=m3)), ((x, x, w), dict(scale=w)),
                     ((x, x, w), dict(scale=m2, shift=m3)), ((x, x, None), dict(h=torch.empty_like(x))), ((x.t(), x.t(), normal((4,), 1).to(dev)), {}), ((x[0], x[0], w), {}),
                     ((x, x, w), dict(y=torch.empty_like(x)[:2]))):
        with pytest.raises(E, match="residual_norm"):
            pkg.residual_norm(*args, **kw)
    pkg.check_cuda_errbuf("after refusals")
    y, h = pkg.residual_norm(x[:0], x[:0], w)
    assert y.shape == h.shape == (0, 64)
    y, _ = pkg.residual_norm(x, x, w, gate=w, scale=m2, shift=m2)
    want, _ = pkg.residual_norm(x, x, w, gate=torch.stack([w, w]), scale=m2, shift=m2)
    assert torch.equal(y, want)


def test_the_entry_point_refuses_before_it_touches_the_gpu(pkg):
    one = C.c_void_p(4096)

    def call(x=one, ldx=8, b=one, ldb=8, post=None, gate=None, pre=one, scale=None, shift=None, groups=1, y=one, ldy=8, h=one, ldh=8, rows=4, cols=8):
        return pkg.lib.o1_residual_norm(x, ldx, b, ldb, post, gate, 1.0, pre, scale, shift, groups, y, ldy, h, ldh, rows, cols, 1e-6)

    for want, args in ((6, dict(x=None)), (6, dict(b=None)), (6, dict(y=None)), (6, dict(pre=None)), (6, dict(scale=one)), (6, dict(shift=one)), (9, dict(rows=-1)),
                       (9, dict(cols=0)), (9, dict(groups=0)), (9, dict(groups=3)), (9, dict(ldx=7)), (9, dict(ldb=7)), (9, dict(ldy=7)), (9, dict(ldh=7))):
        assert call(**args) == want, args
        assert b"residual_norm" in pkg.lib.hd_cuda_last_error()
    assert call(rows=0) == 0
    pkg.lib.hd_cuda_clear_error()


@gpu
@pytest.mark.parametrize("cols", [1152, 4096, 1001])
@pytest.mark.parametrize("eps", [0.0, 1e-37])
def test_small_rows_and_eps(pkg, dev, cols, eps):
    """Rows down to 2^-110 with little or no eps: their squares have no place in 32 bits."""
    f = torch.tensor([1.0, 2.0 ** -40, 2.0 ** -66, 2.0 ** -75, 2.0 ** -110])[:, None]
    x, b = (normal((5, cols), 1).float() * f).to(torch.bfloat16), (normal((5, cols), 2).float() * f).to(torch.bfloat16)
    pre, post = normal((cols,), 3, 0.1), normal((cols,), 4, 0.1)
    y, h = pkg.residual_norm(x.to(dev), b.to(dev), pre.to(dev), post_w=post.to(dev), eps=eps)
    ry, rh, ty, th = reference(x, b, pre, post, None, None, None, 1.0, eps)
    between(y, ry, ty + 1e-45, "y")
    between(h, rh, th + 1e-45, "h")
    y, h = pkg.residual_norm(x.to(dev), b.to(dev), pre.to(dev), eps=eps)
    ry, rh, ty, th = reference(x, b, pre, None, None, None, None, 1.0, eps)
    between(y, ry, ty + 1e-45, "y, no inner norm")
    between(h, rh, th + 1e-45, "h, no inner norm")


@gpu
def test_the_most_rows(pkg, dev):
    """As many rows as an int counts, four to a block (34 GB, in place)."""
    rows = 2 ** 31 - 1
    x = torch.zeros(rows, 8, dtype=torch.bfloat16, device=dev)
    x[-1], x[0] = 1.0, 2.0
    _, h = pkg.residual_norm(x, x, None, y=x)
    assert (x[-1] == 2.0).all() and (x[0] == 4.0).all() and h is None


@gpu
@pytest.mark.parametrize("rows,cols,post,groups", [(1100, 4096, 0, 1), (5003, 4096, 1, 1), (2600, 8192, 1, 2), (600, 8192, 0, 1), (701, 12288, 1, 1), (402, 12288, 0, 2), (1501, 2048, 1, 1),
                                                   (2100, 2048, 0, 3), (10003, 2048, 1, 1), (9001, 1152, 1, 1), (970, 4096, 0, 1), (4800, 4096, 1, 1), (2400, 8192, 1, 1), (400, 8192, 0, 1),
                                                   (640, 12288, 1, 2), (310, 12288, 0, 1)])
def test_many_rows(pkg, dev, rows, cols, post, groups):
    """Sizes beyond which a row has fewer registers and vectors are asked for where they are used, on both sides of each."""
    g = torch.Generator(device=dev).manual_seed(1)
    n = lambda *s: torch.empty(s, dtype=torch.bfloat16, device=dev).normal_(0, 1, generator=g)  # noqa: E731
    x, b, pre, pw = n(rows, cols), n(rows, cols), n(cols), n(cols) if post else None
    gate, scale, shift = n(groups, cols), n(groups, cols), n(groups, cols)
    y, h = pkg.residual_norm(x, b, pre, post_w=pw, gate=gate, scale=scale, shift=shift, alpha=0.4)
    ry, rh, ty, th = reference(x, b, pre, pw, gate, scale, shift, 0.4, 1e-6)
    for got, ref, tol, name in ((y, ry, ty, "y"), (h, rh, th, "h")):
        got = got.double()
        ok = (got >= (ref - tol).to(torch.bfloat16).double()) & (got <= (ref + tol).to(torch.bfloat16).double())
        assert ok.all(), name
    y2, none = pkg.residual_norm(x, b, None, post_w=pw, gate=gate, alpha=0.4)
    assert none is None and torch.equal(y, y2)
