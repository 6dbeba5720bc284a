"""GPU: RMS norm of a residual sum (forward, 8-bit output, backward), the gated feed-forward block (forward, backward) and the linear layer
in 8-bit integers, against the formulas in 64 bits.

Tolerances.  HALF is the half step of a rounding to the type (fp16 2^-11, fp32 2^-24), U = 2^-24 that of the 32-bit sums.
  * a sum of n terms in 32 bits with chains of at most n / 64 terms and a tree above them is off by at most (n / 64 + 16) U times the
    sum of the magnitudes; the element-wise bounds of the norms are these, plus the result's own rounding;
  * the block's products sum on tensor cores whose accumulators truncate.  Their error is held in the 2-norm, where independent roundings add
    in squares: HALF for the result and for each tensor rounded in between, and PRODUCT for the sums: fp16 products of K terms in steps
    of 16, each cut by 2^-23 of a partial sum that grows as sqrt(k): K / 16 * 2^-23 / 4; single precision in three parts, 3 * 2^-22 for what
    the parts leave out, and chains of at most 32 steps cut likewise, or K additions rounded: 0.5 sqrt(K) U.  An element may be eight times as far
    off as that is of the tensor's root mean square;
  * the integer sums are exact: two products with scales, one sum with the bias and the conversion, each one rounding.
"""
import ctypes

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu
U = 2.0 ** -24
HALF = {torch.float16: 2.0 ** -11, torch.float32: 2.0 ** -24}
TINY = {torch.float16: 2.0 ** -25, torch.float32: 0.0}                 # half a step of the smallest numbers
NAME = {torch.float16: "fp16", torch.float32: "fp32"}
EPS = 1e-5
both = pytest.mark.parametrize("dt", [torch.float32, torch.float16], ids=["fp32", "fp16"])


class Ops(object):
    def __init__(self, pkg, lib):
        self.pkg, self.lib = pkg, lib

    def call(self, name, struct, sync=True, **fields):
        """one entry-point call on tensors (device or host), torch's work before and after it in order"""
        keep = self.pkg.Keep()
        args = self.pkg.make_args(keep, "trainlib_%s_args" % struct, **{k: v.data_ptr() if isinstance(v, torch.Tensor) else v for k, v in fields.items()})
        if sync:
            torch.cuda.synchronize()
        getattr(self.lib, "trainlib_" + name)(ctypes.byref(args))
        if sync:
            self.lib.trainlib_synchronize()
            self.pkg.check(self.lib)

    def norm_fw(self, x, res, w, total, y, **kw):
        self.call("rmsnorm_%s_fw_cl" % NAME[x.dtype], "rmsnorm", x=x, residual=res, weight=w, sum=total, output=y, eps=EPS, rows=x.shape[0], size=x.shape[1], **kw)

    def norm_int8(self, x, res, w, total, q, scale, **kw):
        self.call("rmsnorm_int8_%s_fw_cl" % NAME[x.dtype], "rmsnorm", x=x, residual=res, weight=w, sum=total, q=q, scale=scale, eps=EPS, rows=x.shape[0], size=x.shape[1], **kw)

    def norm_bw(self, h, w, dy, dsum, dx, dw, **kw):
        self.call("rmsnorm_%s_bw_cl" % NAME[h.dtype], "rmsnorm", sum=h, weight=w, dy=dy, dsum=dsum, dx=dx, dweight=dw, eps=EPS, rows=h.shape[0], size=h.shape[1], **kw)

    def rows_int8(self, x, q, scale, **kw):
        self.call("quantize_rows_%s_cl" % NAME[x.dtype], "quantize_rows", x=x, q=q, scale=scale, rows=x.shape[0], size=x.shape[1], **kw)

    def linear_int8(self, x, xs, w, ws, bias, y, **kw):
        self.call("linear_int8_%s_fw_cl" % NAME[y.dtype], "linear_int8", x=x, x_scale=xs, weight=w, w_scale=ws, bias=bias, y=y, rows=x.shape[0], in_size=x.shape[1], out_size=w.shape[0], **kw)

    def ffn_fw(self, x, wg, wu, wd, g, u, y, **kw):
        self.call("gated_ffn_%s_fw_cl" % NAME[x.dtype], "gated_ffn", x=x, w_gate=wg, w_up=wu, w_down=wd, gate=g, up=u, y=y,
                  rows=x.shape[0], in_size=x.shape[1], hidden=wg.shape[0], out_size=wd.shape[0], **kw)

    def ffn_bw(self, x, wg, wu, wd, g, u, dy, dx, dwg, dwu, dwd, sizes=None, **kw):
        r, n, h, m = sizes or (x.shape[0], x.shape[1], wg.shape[0], wd.shape[0])
        self.call("gated_ffn_%s_bw_cl" % NAME[dy.dtype], "gated_ffn", x=x, w_gate=wg, w_up=wu, w_down=wd, gate=g, up=u, dy=dy, dx=dx, dw_gate=dwg, dw_up=dwu, dw_down=dwd,
                  rows=r, in_size=n, hidden=h, out_size=m, **kw)


@pytest.fixture
def ops(pkg, gpulib):
    gpulib.trainlib_set_streams(1)
    gpulib.trainlib_set_memory_mode(pkg.TL_MEM_AUTO)
    gpulib.trainlib_set_gemm_path(0)
    return Ops(pkg, gpulib)


def randn(seed, *shape, scale=1.0, dt=torch.float32, shift=0):
    """seeded values; shift: elements between an aligned address and the tensor's"""
    gen = torch.Generator("cuda").manual_seed(seed)
    v = (torch.randn(shape, device="cuda", generator=gen) * scale).to(dt)
    if shift:
        room = torch.empty(v.numel() + shift, device="cuda", dtype=dt)
        room[shift:] = v.reshape(-1)
        v = room[shift:].view(*shape)
    return v


def blank(*shape, dt=torch.float32, shift=0):
    room = torch.full((int(np.prod(shape)) + shift,), 77, device="cuda", dtype=dt)
    return room[shift:].view(*shape)


def within(got, want, bound, what):
    """element by element"""
    far = (got.double() - want).abs() - bound
    assert torch.isfinite(got.double()).all(), what
    assert far.max().item() <= 0, "%s: %g beyond its bound of %g" % (what, far.max().item(), (bound.expand_as(far) if isinstance(bound, torch.Tensor) else torch.tensor(bound)).flatten()[far.argmax().item() if isinstance(bound, torch.Tensor) else 0].item())


# ------------------------------------------------------------------------------------------------ RMS norm
NORMS = [(1, 1), (1, 17), (3, 64), (5, 1000), (2, 4096), (7, 8191), (1, 40000), (300, 256), (33, 130), (64, 1024), (3, 16384), (129, 2048), (1000, 96), (2, 5), (40, 6144), (17, 12345)]


def norm_ref(h, w):
    r = 1 / ((h * h).mean(1, keepdim=True) + EPS).sqrt()
    return h * r * w, r


@both
@pytest.mark.parametrize("shift", [0, 1])
@pytest.mark.parametrize("rows,size", NORMS)
def test_norm_forward(ops, rows, size, shift, dt):
    x, res, w = randn(1, rows, size, dt=dt, shift=shift), randn(2, rows, size, scale=3, dt=dt, shift=shift), (1 + randn(3, size, scale=0.3)).to(dt)
    h = x.double() + res.double()
    want, r = norm_ref(h, w.double())
    chain = (size / 64 + 16) * U
    for residual, keep in ((res, True), (res, False), (None, True)):
        hh, yy = (h, want) if residual is not None else (x.double(), norm_ref(x.double(), w.double())[0])
        total, y = blank(rows, size, dt=dt, shift=shift) if keep else None, blank(rows, size, dt=dt, shift=shift)
        ops.norm_fw(x, residual, w, total, y)
        within(y, yy, yy.abs() * (HALF[dt] + chain) + TINY[dt], "norm")
        if keep:
            within(total, hh, hh.abs() * (HALF[dt] + U) + TINY[dt], "sum")


@both
@pytest.mark.parametrize("shift", [0, 1])
@pytest.mark.parametrize("rows,size", NORMS)
def test_norm_in_8_bits(ops, rows, size, shift, dt):
    x, res, w = randn(4, rows, size, dt=dt, shift=shift), randn(5, rows, size, scale=3, dt=dt, shift=shift), (1 + randn(6, size, scale=0.3)).to(dt)
    h = x.double() + res.double()
    want, r = norm_ref(h, w.double())
    total, q, scale = blank(rows, size, dt=dt, shift=shift), blank(rows, size, dt=torch.int8, shift=shift), blank(rows)
    ops.norm_int8(x, res, w, total, q, scale)
    step = want.abs().amax(1) / 127
    within(scale, step, step * (size / 64 + 16) * U, "scale")
    # half a step, and what eight roundings of a value of up to 127 steps move it
    within(q, want / step[:, None], 0.5 + 127 * 8 * U, "q")
    assert (q.abs().amax(1) == 127).all()
    within(total, h, h.abs() * (HALF[dt] + U) + TINY[dt], "sum")
    ops.rows_int8(x, q, scale)
    step = x.double().abs().amax(1) / 127
    within(scale, step, step * 2 * U, "scale of the rows")
    within(q, x.double() / step[:, None], 0.5 + 127 * 4 * U, "q of the rows")


@both
@pytest.mark.parametrize("rows,size", NORMS + [(2000, 40), (4100, 512), (513, 2176), (700, 331), (1300, 499), (40, 510)])
def test_norm_backward(ops, rows, size, dt):
    for shift in (0, 1):
        h, dy, dsum = randn(7, rows, size, scale=2, dt=dt, shift=shift), randn(8, rows, size, dt=dt, shift=shift), randn(9, rows, size, dt=dt, shift=shift)
        w = (1 + randn(10, size, scale=0.3)).to(dt)
        hd, wd = h.double().requires_grad_(), w.double().requires_grad_()
        want_dx, want_dw = torch.autograd.grad(norm_ref(hd, wd)[0], [hd, wd], dy.double())
        _, r = norm_ref(h.double(), w.double())
        g = (dy.double() * w.double()).abs()
        scale = r * g + h.double().abs() * r ** 3 * (g * h.double().abs()).mean(1, keepdim=True)
        terms = (dy.double() * h.double() * r).abs().sum(0)
        for plus in (dsum, None):
            full = want_dx + plus.double() if plus is not None else want_dx
            dx, dw = blank(rows, size, dt=dt, shift=shift), blank(size, dt=dt)
            ops.norm_bw(h, w, dy, plus, dx, dw)
            within(dx, full, full.abs() * HALF[dt] + ((plus.double().abs() if plus is not None else 0) + scale) * (size / 64 + 16) * U + TINY[dt], "dx")
            within(dw, want_dw, want_dw.abs() * HALF[dt] + terms * (rows / 32 + size / 64 + 128) * U + TINY[dt], "dweight")
        only = blank(rows, size, dt=dt, shift=shift)
        ops.norm_bw(h, w, dy, None, only, None)
        assert torch.equal(only, dx)
        alone = blank(size, dt=dt)
        ops.norm_bw(h, w, dy, None, None, alone)
        assert torch.equal(alone, dw)


@both
@pytest.mark.parametrize("rows,size", [(3, 64), (5, 1001), (2, 4096), (3, 40000), (600, 512)])
def test_norm_in_place(ops, rows, size, dt):
    """the sum and the norm may be written over x or the residual, the gradient over any of its inputs"""
    x, res, w = randn(11, rows, size, dt=dt), randn(12, rows, size, dt=dt), (1 + randn(13, size, scale=0.3)).to(dt)
    total, y = blank(rows, size, dt=dt), blank(rows, size, dt=dt)
    ops.norm_fw(x, res, w, total, y)
    a, b = x.clone(), res.clone()
    ops.norm_fw(a, b, w, b, a)
    assert torch.equal(a, y) and torch.equal(b, total)
    a, b = x.clone(), res.clone()
    ops.norm_fw(a, b, w, a, b)
    assert torch.equal(b, y) and torch.equal(a, total)
    q, scale, q2, s2 = blank(rows, size, dt=torch.int8), blank(rows), blank(rows, size, dt=torch.int8), blank(rows)
    ops.norm_int8(x, res, w, None, q, scale)
    b = res.clone()
    ops.norm_int8(x, b, w, b, q2, s2)
    assert torch.equal(b, total) and torch.equal(q, q2) and torch.equal(scale, s2)
    dy, dsum = randn(14, rows, size, dt=dt), randn(15, rows, size, dt=dt)
    dx, dw = blank(rows, size, dt=dt), blank(size, dt=dt)
    ops.norm_bw(total, w, dy, dsum, dx, dw)
    for at in range(3):
        ins = [total.clone(), dy.clone(), dsum.clone()]
        dw2 = blank(size, dt=dt)
        ops.norm_bw(ins[0], w, ins[1], ins[2], ins[at], dw2)
        assert torch.equal(ins[at], dx) and torch.equal(dw2, dw)


@both
@pytest.mark.parametrize("size", [5, 96, 1000, 4096, 40000])
def test_norm_rows_of_zeros_and_of_no_numbers(ops, size, dt):
    """a row of zeros, one with an infinity, one with a NaN and rows of tiny values: the others stay as they are"""
    rows = 9
    x, w = randn(16, rows, size, dt=dt), (1 + randn(17, size, scale=0.3)).to(dt)
    clean_y, clean_q, clean_s = blank(rows, size, dt=dt), blank(rows, size, dt=torch.int8), blank(rows)
    ops.norm_fw(x, None, w, None, clean_y)
    ops.norm_int8(x, None, w, None, clean_q, clean_s)
    v = x.clone()
    v[1] = 0
    v[3, size // 2] = float("inf")
    v[5, size - 1] = float("nan")
    v[7] = v[7] * 2.0 ** -12
    y, q, s = blank(rows, size, dt=dt), blank(rows, size, dt=torch.int8), blank(rows)
    ops.norm_fw(v, None, w, None, y)
    ops.norm_int8(v, None, w, None, q, s)
    same = [0, 2, 4, 6, 8]
    assert torch.equal(y[same], clean_y[same]) and torch.equal(q[same], clean_q[same]) and torch.equal(s[same], clean_s[same])
    assert (y[1] == 0).all() and (q[1] == 0).all() and s[1] == 0
    assert torch.isnan(y[3, size // 2]) and torch.isnan(y[5]).all()
    assert not torch.isfinite(s[3]) and not torch.isfinite(s[5])
    want, _ = norm_ref(v[7:8].double(), w.double())
    within(y[7:8], want, want.abs() * (HALF[dt] + (size / 64 + 16) * U) + TINY[dt], "tiny")
    ops.rows_int8(v, q, s)
    assert (q[1] == 0).all() and s[1] == 0 and not torch.isfinite(s[3]) and not torch.isfinite(s[5])
    if dt == torch.float32:
        # magnitudes whose squares leave 32 bits, and the smallest ones: the 8-bit form of rows does not square them
        for scale in (1e30, 1e-37, 1e-42):
            big = (x.double() * scale).float()
            ops.rows_int8(big, q, s)
            step = big.double().abs().amax(1) / 127
            within(s, step, step * 2 * U + 2.0 ** -149, "scale")
            within(q, big.double() / step[:, None], 0.5 + 127 * 4 * U, "q")


@both
def test_norm_gradient_against_differences(ops, dt):
    """<gradient, direction> against the forward pass at two points on either side of it.  The forward pass in 32 bits: its rounding of 2^-23 of
    values of up to 4 over a step of 2^-6 and a sum of rows * size random terms; the second-order term is 2^-12 of the third derivative."""
    if dt == torch.float16:
        pytest.skip("steps of half precision are as large as the differences")
    rows, size = 6, 200
    h, w, dy = randn(18, rows, size), 1 + randn(19, size, scale=0.3), randn(20, rows, size)
    dx, dw = blank(rows, size), blank(size)
    ops.norm_bw(h, w, dy, None, dx, dw)
    d, e, step = randn(21, rows, size), randn(22, size), 2.0 ** -6
    ys = []
    for k in (1, -1):
        y = blank(rows, size)
        ops.norm_fw(h + k * step * d, None, w + k * step * e, None, y)
        ys.append((y.double() * dy.double()).sum())
    got = ((ys[0] - ys[1]) / (2 * step)).item()
    want = ((dx.double() * d.double()).sum() + (dw.double() * e.double()).sum()).item()
    spread = (rows * size) ** 0.5
    assert abs(got - want) <= spread * (4 * 2.0 ** -23 / step + 4 * step ** 2), (got, want)


# ------------------------------------------------------------------------------------------------ linear layer in 8 bits
LINEAR8 = [(1, 1, 1), (1, 64, 32), (2, 17, 5), (3, 100, 1001), (7, 1024, 130), (8, 4096, 512), (9, 260, 64), (16, 512, 777), (17, 128, 128), (33, 1001, 257), (64, 2048, 96), (100, 36, 300),
           (129, 640, 520), (200, 48, 1000), (257, 1008, 129), (333, 1001, 777), (512, 2048, 1024), (1, 8191, 333), (5, 16400, 40), (300, 4112, 200), (1000, 128, 8), (31, 20, 3000)]


@both
@pytest.mark.parametrize("rows,n,m", LINEAR8)
def test_linear_in_8_bits(ops, rows, n, m, dt):
    gen = torch.Generator("cuda").manual_seed(rows + n + m)
    for shift in (0, 1):
        x = blank(rows, n, dt=torch.int8, shift=shift).copy_(torch.randint(-128, 128, (rows, n), device="cuda", generator=gen))
        w = blank(m, n, dt=torch.int8, shift=shift).copy_(torch.randint(-128, 128, (m, n), device="cuda", generator=gen))
        xs, ws = torch.rand(rows, device="cuda", generator=gen) / 127, torch.rand(m, device="cuda", generator=gen) / 127 / n ** 0.5
        bias = randn(23, m, dt=dt)
        product = (x.double() @ w.double().T) * xs.double()[:, None] * ws.double()
        for b in (bias, None):
            y = blank(rows, m, dt=dt, shift=shift)
            ops.linear_int8(x, xs, w, ws, b, y)
            want = product + b.double() if b is not None else product
            within(y, want, product.abs() * 3 * U * 1.01 + want.abs() * (U + HALF[dt]) * 1.01 + TINY[dt], "y")


@both
def test_linear_in_8_bits_at_the_ends_of_the_range(ops, dt):
    """sums of the largest magnitude that 32 bits hold, and scales that are zero or no numbers"""
    n = 131071
    x, w = torch.full((3, n), -128, dtype=torch.int8, device="cuda"), torch.full((5, n), -128, dtype=torch.int8, device="cuda")
    w[1] = 127
    xs, ws = torch.tensor([2.0 ** -20, 0.0, float("nan")], device="cuda"), torch.full((5,), 2.0 ** -8, device="cuda")
    y = blank(3, 5, dt=dt)
    ops.linear_int8(x, xs, w, ws, None, y)
    want = (x[:1].double() @ w.double().T) * 2.0 ** -28
    within(y[:1], want, want.abs() * (U + HALF[dt]) * 1.01, "largest sums")
    assert (y[1] == 0).all() and torch.isnan(y[2]).all()


# ------------------------------------------------------------------------------------------------ gated feed-forward block
FFNS = [(1, 1, 1, 1), (1, 64, 96, 64), (3, 17, 33, 5), (2, 1024, 512, 256), (8, 256, 1000, 256), (9, 72, 200, 1), (23, 1000, 2731, 1000), (33, 512, 136, 520), (64, 128, 256, 64), (130, 257, 129, 63),
        (128, 512, 512, 512), (300, 264, 520, 136), (257, 640, 1096, 384), (512, 1024, 1000, 512), (1, 2500, 3000, 1001), (1030, 192, 392, 200), (16, 2048, 640, 2048), (1, 8, 5000, 8), (700, 8, 16, 8)]


def silu(v):
    return v / (1 + torch.exp(-v))


def product_error(dt, *lengths):
    """2-norm error of sums over products of these lengths, one behind the other"""
    if dt == torch.float16:
        return sum(k / 16 * 2.0 ** -23 / 4 + 2.0 ** -22 for k in lengths)
    return sum(3 * 2.0 ** -22 + 32 * 2.0 ** -23 / 4 + 0.5 * k ** 0.5 * U for k in lengths)


def near(got, want, dt, roundings, products, what, terms=None):
    """2-norm: `roundings` independent roundings to the type, one the result's; sums over `products`; elements: the half step and eight times the rest.
    terms: for each result the sum of the squares of the terms a * b that it adds.  Roundings of the a, each d_k |a_k| with independent |d_k| <= HALF, move
    the result by sum d_k a_k b_k, whose mean square is at most HALF^2 / 3 * sum (a_k b_k)^2: that, and not the result, is what their bound is
    relative to.  Over many results the two agree (terms of random sign); of fifteen results of 33 terms the results' squares may add up to less."""
    assert torch.isfinite(got.double()).all(), what
    off, rms = got.double() - want, want.square().mean().sqrt()
    if terms is not None:
        rms = torch.maximum(rms, terms.mean().sqrt())
    tol = HALF[dt] * roundings ** 0.5 + product_error(dt, *products)
    norm = off.square().mean().sqrt()
    assert norm <= tol * rms + TINY[dt], "%s: %g of %g allowed" % (what, norm / rms, tol)
    # An element's share of those roundings is relative to the root of its own terms' squares (for the single term of an outer product, to that term),
    # which may be many times the tensor's root mean square where two large factors meet.
    own = terms.sqrt() if terms is not None else rms
    worst = (off.abs() - want.abs() * HALF[dt] - 8 * HALF[dt] * (roundings - 1) ** 0.5 * own).max()
    assert worst <= 8 * product_error(dt, *products) * rms + TINY[dt], "%s: an element %g of %g allowed" % (what, worst / rms, 8 * product_error(dt, *products))


def ffn_tensors(rows, n, h, m, dt, shift=0, seed=30):
    return (randn(seed, rows, n, dt=dt, shift=shift), randn(seed + 1, h, n, scale=n ** -0.5, dt=dt, shift=shift), randn(seed + 2, h, n, scale=n ** -0.5, dt=dt, shift=shift),
            randn(seed + 3, m, h, scale=h ** -0.5, dt=dt, shift=shift))


@both
@pytest.mark.parametrize("rows,n,h,m", FFNS)
def test_ffn_forward(ops, rows, n, h, m, dt):
    for shift in (0, 1):
        x, wg, wu, wd = ffn_tensors(rows, n, h, m, dt, shift)
        gd, ud = x.double() @ wg.double().T, x.double() @ wu.double().T
        want = (silu(gd) * ud) @ wd.double().T
        terms = (silu(gd) * ud).square() @ wd.double().square().T
        y, g, u = blank(rows, m, dt=dt, shift=shift), blank(rows, h, dt=dt, shift=shift), blank(rows, h, dt=dt, shift=shift)
        ops.ffn_fw(x, wg, wu, wd, g, u, y)
        near(y, want, dt, 2, (3 * n, h), "y", terms)             # (G, U and silu's argument: three of the first products' errors)
        near(g, gd, dt, 1, (n,), "gate")
        near(u, ud, dt, 1, (n,), "up")
        y2 = blank(rows, m, dt=dt, shift=shift)
        ops.ffn_fw(x, wg, wu, wd, None, None, y2)
        assert torch.equal(y, y2)


def ffn_bw_ref(x, wg, wu, wd, g, u, dy):
    g, u, wd = g.double().requires_grad_(), u.double().requires_grad_(), wd.double().requires_grad_()
    dg, du, dwd = torch.autograd.grad((silu(g) * u) @ wd.T, [g, u, wd], dy.double())
    sq = lambda t: t.detach().double().square()  # noqa: E731
    return ((dg @ wg.double() + du @ wu.double(), dg.T @ x.double(), du.T @ x.double(), dwd),
            (sq(dg) @ sq(wg) + sq(du) @ sq(wu), sq(dg).T @ sq(x), sq(du).T @ sq(x), sq(dy).T @ sq(silu(g) * u)))


@both
@pytest.mark.parametrize("rows,n,h,m", FFNS)
def test_ffn_backward(ops, rows, n, h, m, dt):
    for shift in (0, 1):
        x, wg, wu, wd = ffn_tensors(rows, n, h, m, dt, shift)
        g, u, dy = randn(40, rows, h, dt=dt, shift=shift), randn(41, rows, h, dt=dt, shift=shift), randn(42, rows, m, dt=dt, shift=shift)
        want, terms = ffn_bw_ref(x, wg, wu, wd, g, u, dy)
        got = [blank(*t.shape, dt=dt, shift=shift) for t in (x, wg, wu, wd)]
        ops.ffn_bw(x, wg, wu, wd, g, u, dy, *got)
        for t, v, q, k, what in zip(got, want, terms, (2 * h, rows, rows, rows), ("dx", "dw_gate", "dw_up", "dw_down")):
            near(t, v, dt, 2, (m, k), what, q)
        # every gradient on its own, without the operands that it does not need
        alone = [blank(*t.shape, dt=dt, shift=shift) for t in (x, wg, wu, wd)]
        s = (rows, n, h, m)
        ops.ffn_bw(None, wg, wu, wd, g, u, dy, alone[0], None, None, None, sizes=s)
        ops.ffn_bw(x, None, None, wd, g, u, dy, None, alone[1], None, None, sizes=s)
        ops.ffn_bw(x, None, None, wd, g, u, dy, None, None, alone[2], None, sizes=s)
        ops.ffn_bw(None, None, None, None, g, u, dy, None, None, None, alone[3], sizes=s)
        # (a launch of all of them may share a sum's terms out differently: the same bounds, not the same bits)
        for t, v, q, k, what in zip(alone, want, terms, (2 * h, rows, rows, rows), ("dx", "dw_gate", "dw_up", "dw_down")):
            near(t, v, dt, 2, (m, k), what + " alone", q)


@pytest.mark.parametrize("rows,n,h,m", [(4100, 136, 8200, 2048), (4096, 2048, 2056, 1000), (2300, 1032, 8192, 264), (4100, 136, 8199, 2050)])
def test_ffn_of_many_tiles(ops, rows, n, h, m):
    """sizes whose products run on pairs of CTAs, some with rows and columns behind the last whole tile, some that are not read in place"""
    dt = torch.float16
    x, wg, wu, wd = ffn_tensors(rows, n, h, m, dt)
    gd, ud = x.double() @ wg.double().T, x.double() @ wu.double().T
    want, terms = (silu(gd) * ud) @ wd.double().T, (silu(gd) * ud).square() @ wd.double().square().T
    y, g, u = blank(rows, m, dt=dt), blank(rows, h, dt=dt), blank(rows, h, dt=dt)
    ops.ffn_fw(x, wg, wu, wd, g, u, y)
    near(y, want, dt, 2, (3 * n, h), "y", terms)
    near(g, gd, dt, 1, (n,), "gate")
    near(u, ud, dt, 1, (n,), "up")
    dy = randn(42, rows, m, dt=dt)
    want, terms = ffn_bw_ref(x, wg, wu, wd, g, u, dy)
    room = [torch.full((t.numel() + 4096,), 77, device="cuda", dtype=dt) for t in (x, wg, wu, wd)]
    got = [r[:t.numel()].view_as(t) for r, t in zip(room, (x, wg, wu, wd))]
    ops.ffn_bw(x, wg, wu, wd, g, u, dy, *got)
    for t, v, q, k, what in zip(got, want, terms, (2 * h, rows, rows, rows), ("dx", "dw_gate", "dw_up", "dw_down")):
        near(t, v, dt, 2, (m, k), what, q)
    assert all((r[t.numel():] == 77).all() for r, t in zip(room, got))
    again = [blank(*t.shape, dt=dt) for t in got]
    ops.ffn_bw(x, wg, wu, wd, g, u, dy, *again)
    assert all(torch.equal(a, b) for a, b in zip(again, got))


@both
@pytest.mark.parametrize("rows", [1, 9, 20, 32])
def test_ffn_few_tokens_of_odd_widths(ops, rows, dt):
    """rows that start between two groups of sixteen bytes and end around a whole number of what the warps take at a time, in the first products and in the last"""
    for k in (127, 131, 257, 511, 513, 545, 1025, 1027, 2050, 2731):
        for n, h in ((k, 24), (40, k)):
            for shift in (0, 2):
                x, wg, wu, wd = ffn_tensors(rows, n, h, 33, dt, shift, seed=50 + k)
                gd, ud = x.double() @ wg.double().T, x.double() @ wu.double().T
                y = blank(rows, 33, dt=dt)
                ops.ffn_fw(x, wg, wu, wd, None, None, y)
                near(y, (silu(gd) * ud) @ wd.double().T, dt, 2, (3 * n, h), "y", (silu(gd) * ud).square() @ wd.double().square().T)


@pytest.mark.parametrize("rows", [1, 9, 20, 32, 33, 150])
def test_linear_in_8_bits_of_odd_widths(ops, rows):
    """whole numbers: the sums are exact and rounded once"""
    gen = torch.Generator("cuda").manual_seed(rows)
    for k in (515, 1023, 1025, 1026, 1087, 1089, 2113, 4099):
        for shift in (0, 1, 4):
            x = blank(rows, k, dt=torch.int8, shift=shift).copy_(torch.randint(-128, 128, (rows, k), device="cuda", generator=gen))
            w = blank(37, k, dt=torch.int8, shift=shift).copy_(torch.randint(-128, 128, (37, k), device="cuda", generator=gen))
            y = blank(rows, 37)
            ops.linear_int8(x, torch.ones(rows, device="cuda"), w, torch.ones(37, device="cuda"), None, y)
            assert torch.equal(y, (x.double() @ w.double().T).float()), (k, shift)


@both
def test_ffn_rows_of_no_numbers_stay_apart(ops, dt):
    for rows, n, h, m in ((3, 64, 96, 40), (200, 256, 384, 128), (300, 100, 70, 50)):
        x, wg, wu, wd = ffn_tensors(rows, n, h, m, dt)
        y, g, u = blank(rows, m, dt=dt), blank(rows, h, dt=dt), blank(rows, h, dt=dt)
        ops.ffn_fw(x, wg, wu, wd, g, u, y)
        v = x.clone()
        v[1, 5], v[rows - 1, n - 1] = float("nan"), float("inf")
        y2, g2, u2 = blank(rows, m, dt=dt), blank(rows, h, dt=dt), blank(rows, h, dt=dt)
        ops.ffn_fw(v, wg, wu, wd, g2, u2, y2)
        fine = torch.ones(rows, dtype=torch.bool)
        fine[1] = fine[rows - 1] = False
        assert torch.equal(y[fine], y2[fine]) and torch.isnan(y2[1]).all() and not torch.isfinite(y2[rows - 1].float()).any() and torch.isnan(g2[1]).all()
        dy = randn(43, rows, m, dt=dt)
        dx, dx2 = blank(rows, n, dt=dt), blank(rows, n, dt=dt)
        ops.ffn_bw(x, wg, wu, wd, g, u, dy, dx, None, None, None)
        ops.ffn_bw(x, wg, wu, wd, g2, u2, dy, dx2, None, None, None)
        assert torch.equal(dx[fine], dx2[fine]) and torch.isnan(dx2[1]).all()


def test_gate_at_the_ends_of_its_range(ops):
    """gates far from zero: silu tends to v and to 0, its derivative to 1 and 0, without a NaN on the way"""
    for dt, far in ((torch.float32, 1e4), (torch.float16, 6e4)):
        rows, h = 4, 24
        g, u, dy = blank(rows, h, dt=dt), randn(44, rows, h, dt=dt), randn(45, rows, h, dt=dt)
        g[:, :12], g[:, 12:] = far, -far
        g[0, 0], g[0, 23] = 90.0, -90.0
        wd = torch.eye(h, device="cuda").to(dt)
        one = torch.eye(h, device="cuda").to(dt)
        dx = blank(rows, h, dt=dt)
        zero = torch.zeros(h, h, device="cuda", dtype=dt)
        ops.ffn_bw(None, one, zero, wd, g, u, dy, dx, None, None, None, sizes=(rows, h, h, h))
        want = torch.where(g > 0, dy.double() * u.double(), torch.zeros(rows, h, device="cuda", dtype=torch.float64))
        # dU = dH silu(G) is held in the type between the products: beyond 65504 + half a step (65520) it is infinite in half precision, and its row of
        # dX, which adds 0 * dU here, is NaN
        over = (dy.double() * g.double().clamp(min=0)).abs().amax(1) >= (65520 if dt == torch.float16 else float("inf"))
        assert torch.isnan(dx[over]).all() and not over.all()
        dx, want = dx[~over], want[~over]
        within(dx, want, want.abs() * (2 * HALF[dt] + 8 * U) + 1e-30 + TINY[dt], "dgate")


def test_ffn_gradients_against_differences(ops):
    """single precision: <gradients, directions> against the forward pass on either side; steps of 2^-7, values of order 1, so 2^-14 of the third
    derivative's and 2^-21 / 2^-7 of the products' error, times the root of the number of terms"""
    rows, n, h, m = 9, 48, 80, 40
    ts = ffn_tensors(rows, n, h, m, torch.float32)
    dy, y, g, u = randn(46, rows, m), blank(rows, m), blank(rows, h), blank(rows, h)
    ops.ffn_fw(*ts, g, u, y)
    grads = [blank(*t.shape) for t in ts]
    ops.ffn_bw(*ts, g, u, dy, *grads)
    for k, t in enumerate(ts):
        d, step, sums = randn(47 + k, *t.shape, scale=t.square().mean().sqrt().item()), 2.0 ** -7, []
        for sign in (1, -1):
            moved = [v + sign * step * d if j == k else v for j, v in enumerate(ts)]
            ops.ffn_fw(*moved, None, None, y)
            sums.append((y.double() * dy.double()).sum())
        got, want = ((sums[0] - sums[1]) / (2 * step)).item(), (grads[k].double() * d.double()).sum().item()
        assert abs(got - want) <= (rows * m) ** 0.5 * (4 * step ** 2 + 2.0 ** -21 / step), (k, got, want)


# ------------------------------------------------------------------------------------------------ together, as they are used
@both
def test_training_block(ops, dt):
    """sum and norm, feed-forward block, sum and norm; back through all of them, against differentiation of the whole in 64 bits"""
    rows, n, h = 150, 256, 640
    x, res = randn(60, rows, n, dt=dt), randn(61, rows, n, dt=dt)
    w1, w2 = (1 + randn(62, n, scale=0.2)).to(dt), (1 + randn(63, n, scale=0.2)).to(dt)
    _, wg, wu, wd = ffn_tensors(rows, n, h, n, dt, seed=64)
    new = lambda *s: blank(*s, dt=dt)  # noqa: E731
    h1, y1, g, u, f, h2, y2 = new(rows, n), new(rows, n), new(rows, h), new(rows, h), new(rows, n), new(rows, n), new(rows, n)
    ops.norm_fw(x, res, w1, h1, y1)
    ops.ffn_fw(y1, wg, wu, wd, g, u, f)
    ops.norm_fw(f, h1, w2, h2, y2)
    dy2 = randn(70, rows, n, dt=dt)
    dh2, dw2, dy1, dwg, dwu, dwd, dh1, dw1 = new(rows, n), new(n), new(rows, n), new(h, n), new(h, n), new(n, h), new(rows, n), new(n)
    ops.norm_bw(h2, w2, dy2, None, dh2, dw2)
    ops.ffn_bw(y1, wg, wu, wd, g, u, dh2, dy1, dwg, dwu, dwd)
    ops.norm_bw(h1, w1, dy1, dh2, dh1, dw1)
    leaves = [t.double().requires_grad_() for t in (x, w1, wg, wu, wd, w2)]
    X, W1, WG, WU, WD, W2 = leaves
    H1 = X + res.double()
    Y1 = norm_ref(H1, W1)[0]
    H2 = H1 + (silu(Y1 @ WG.T) * (Y1 @ WU.T)) @ WD.T
    Y2 = norm_ref(H2, W2)[0]
    # at most eight tensors are rounded on the way there and eight on the way back; each product's sums besides
    near(y2, Y2.detach(), dt, 8, (4 * n, 2 * h), "y")
    for got, want, what in zip((dh1, dw1, dwg, dwu, dwd, dw2), torch.autograd.grad(Y2, leaves, dy2.double()), ("dx", "dw1", "dw_gate", "dw_up", "dw_down", "dw2")):
        near(got, want, dt, 16, (8 * n, 4 * h, 2 * rows), what)


@both
@pytest.mark.parametrize("rows", [1, 5, 40, 260])
def test_serving_block_in_8_bits(ops, rows, dt):
    """norm in 8 bits, both projections in 8 bits, the framework's SwiGLU, its rows in 8 bits, the projection back: against the same in 64 bits.
    The quantisation of either side picks the same step but beside a border, where the neighbouring one moves a result by 2^-7 / sqrt(width) of its size."""
    n, h = 320, 704
    x, res, w = randn(80, rows, n, dt=dt), randn(81, rows, n, dt=dt), (1 + randn(82, n, scale=0.2)).to(dt)
    ws = [randn(83 + k, *s, scale=s[1] ** -0.5) for k, s in enumerate(((h, n), (h, n), (n, h)))]
    q8 = [(blank(*t.shape, dt=torch.int8), blank(t.shape[0])) for t in ws]
    for t, (q, s) in zip(ws, q8):
        ops.rows_int8(t, q, s)
    total, q, s = blank(rows, n, dt=dt), blank(rows, n, dt=torch.int8), blank(rows)
    g, u, a, y = blank(rows, h, dt=dt), blank(rows, h, dt=dt), blank(rows, h, dt=dt), blank(rows, n, dt=dt)
    ops.norm_int8(x, res, w, total, q, s)
    ops.linear_int8(q, s, *q8[0], None, g)
    ops.linear_int8(q, s, *q8[1], None, u)
    keep = ops.pkg.Keep()
    ops.pkg.call(ops.lib, "pulp_swiglu_%s_cl" % NAME[dt], ops.pkg.make_args(keep, "swiglu_args" + ("_fp16" if dt == torch.float16 else ""), in1=g.data_ptr(), in2=u.data_ptr(), out=a.data_ptr(), dim=rows * h))
    qa, sa = blank(rows, h, dt=torch.int8), blank(rows)
    ops.rows_int8(a, qa, sa)
    ops.linear_int8(qa, sa, *q8[2], None, y)

    def quantised(v):
        step = v.abs().amax(1, keepdim=True) / 127
        return (v / step).round() * step
    W = [q.double() * s.double()[:, None] for q, s in q8]
    Y = quantised(norm_ref(x.double() + res.double(), w.double())[0])
    A = quantised(silu(Y @ W[0].T) * (Y @ W[1].T))
    want = A @ W[2].T
    # a step's rounding of either side differs for the share of values whose neighbourhood of `HALF * 127` steps holds a border
    flips = (2 * 127 * (HALF[dt] * 4 + 16 * U)) ** 0.5 * 2.0 ** -6
    off, rms = (y.double() - want).square().mean().sqrt(), want.square().mean().sqrt()
    assert off <= (4 * HALF[dt] + flips) * rms, off / rms


@both
def test_host_tensors(ops, dt):
    """ordinary host arrays: staged, written back, the same bits as on the device"""
    rows, n, h, m = 37, 96, 120, 72
    x, wg, wu, wd = ffn_tensors(rows, n, h, m, dt)
    res, w, dy = randn(90, rows, n, dt=dt), (1 + randn(91, n, scale=0.2)).to(dt), randn(92, rows, m, dt=dt)
    cpu = lambda *ts: [t.cpu() if t is not None else None for t in ts]  # noqa: E731

    def everything(where):
        ins = [t.to(where) for t in (x, res, w, wg, wu, wd, dy)]
        X, R, W, WG, WU, WD, DY = ins
        z = lambda *s, d=dt: torch.zeros(s, dtype=d, device=where)  # noqa: E731
        total, y, q, s, g, u, f = z(rows, n), z(rows, n), z(rows, n, d=torch.int8), z(rows, d=torch.float32), z(rows, h), z(rows, h), z(rows, m)
        ops.norm_fw(X, R, W, total, y)
        ops.norm_int8(X, R, W, None, q, s)
        ops.ffn_fw(y, WG, WU, WD, g, u, f)
        grads = [z(*t.shape) for t in (X, WG, WU, WD)]
        ops.ffn_bw(y, WG, WU, WD, g, u, DY, *grads)
        dx, dw = z(rows, n), z(n)
        ops.norm_bw(total, W, grads[0], None, dx, dw)
        q8, s8, l8 = z(h, n, d=torch.int8), z(h, d=torch.float32), z(rows, h)
        ops.rows_int8(WG, q8, s8)
        ops.linear_int8(q, s, q8, s8, None, l8)
        return cpu(total, y, q, s, g, u, f, *grads, dx, dw, q8, s8, l8)
    for a, b in zip(everything("cuda"), everything("cpu")):
        assert torch.equal(a, b)


@both
@pytest.mark.parametrize("rows,n,h", [(3, 64, 96), (40, 512, 200), (300, 512, 640), (20, 333, 777), (150, 259, 1001)])
def test_recorded_and_replayed(ops, rows, n, h, dt):
    """two recorded graphs that share the library's scratch, replayed in turn on new inputs: the bits of direct calls"""
    def program(seed):
        x, wg, wu, wd = ffn_tensors(rows, n, h, n, dt, seed=seed)
        w, res, dy = (1 + randn(seed + 5, n, scale=0.2)).to(dt), randn(seed + 6, rows, n, dt=dt), randn(seed + 7, rows, n, dt=dt)
        new = lambda *s, d=dt: blank(*s, dt=d)  # noqa: E731
        t = dict(h=new(rows, n), y=new(rows, n), g=new(rows, h), u=new(rows, h), f=new(rows, n), dx=new(rows, n), dwg=new(h, n), dwu=new(h, n), dwd=new(n, h), dh=new(rows, n), dw=new(n),
                 q=new(rows, n, d=torch.int8), s=new(rows, d=torch.float32), wq=new(h, n, d=torch.int8), wqs=new(h, d=torch.float32), l=new(rows, h))

        def step():
            kw = dict(sync=False)
            ops.norm_fw(x, res, w, t["h"], t["y"], **kw)
            ops.ffn_fw(t["y"], wg, wu, wd, t["g"], t["u"], t["f"], **kw)
            ops.ffn_bw(t["y"], wg, wu, wd, t["g"], t["u"], dy, t["dx"], t["dwg"], t["dwu"], t["dwd"], **kw)
            ops.norm_bw(t["h"], w, t["dx"], dy, t["dh"], t["dw"], **kw)
            ops.norm_int8(x, res, w, None, t["q"], t["s"], **kw)
            ops.rows_int8(wg, t["wq"], t["wqs"], **kw)
            ops.linear_int8(t["q"], t["s"], t["wq"], t["wqs"], None, t["l"], **kw)
        return x, t, step
    progs = [program(100), program(200)]
    graphs = []
    for x, t, step in progs:
        torch.cuda.synchronize()
        step()
        ops.lib.trainlib_synchronize()
    for x, t, step in progs:
        assert ops.lib.trainlib_graph_begin() == 0
        step()
        graphs.append(ops.lib.trainlib_graph_end())
        assert graphs[-1], ops.lib.trainlib_last_error_string()
    for k, (x, t, step) in enumerate(progs):
        x.copy_(randn(300 + k, rows, n, dt=dt))
        for v in t.values():
            v.fill_(1)
    torch.cuda.synchronize()
    for _ in range(2):
        for gr in graphs:
            assert ops.lib.trainlib_graph_launch(gr) == 0
    ops.lib.trainlib_synchronize()
    ops.pkg.check(ops.lib)
    for x, t, step in progs:
        replayed = {k: v.clone() for k, v in t.items()}
        for v in t.values():
            v.fill_(2)
        torch.cuda.synchronize()
        step()
        ops.lib.trainlib_synchronize()
        for k, v in t.items():
            assert torch.equal(v, replayed[k]), k
    for gr in graphs:
        ops.lib.trainlib_graph_destroy(gr)


@both
def test_on_a_stream_of_the_caller(ops, dt):
    """queued on the caller's stream behind the kernel that makes the input, and back on the library's own: the same bits"""
    rows, n, h = 90, 256, 384
    x, wg, wu, wd = ffn_tensors(rows, n, h, n, dt)
    y, y2 = blank(rows, n, dt=dt), blank(rows, n, dt=dt)
    ops.ffn_fw(x, wg, wu, wd, None, None, y)
    side = torch.cuda.Stream()
    torch.cuda.synchronize()
    with torch.cuda.stream(side):
        ops.lib.trainlib_set_stream(side.cuda_stream)
        late = torch.zeros_like(x)
        for _ in range(20):
            late.copy_(x)
        ops.ffn_fw(late, wg, wu, wd, None, None, y2, sync=False)
        got = y2.clone()
    torch.cuda.synchronize()
    ops.lib.trainlib_set_stream(None)
    ops.pkg.check(ops.lib)
    assert torch.equal(got, y)


@both
def test_the_same_bits_every_time_and_nothing_beside_them(ops, dt):
    """results do not depend on the run; rows and columns behind the last are left as they were"""
    for rows, n, h, m in ((5, 520, 264, 72), (200, 264, 200, 392), (1100, 256, 72, 100)):
        x, wg, wu, wd = ffn_tensors(rows, n, h, m, dt)
        w, dy = (1 + randn(110, n, scale=0.2)).to(dt), randn(111, rows, m, dt=dt)
        wq, wqs = blank(h, n, dt=torch.int8), blank(h)
        ops.rows_int8(wg, wq, wqs)
        first = None
        for _ in range(3):
            pad = lambda *s, d=dt: torch.full((int(np.prod(s)) + 4096,), 77, device="cuda", dtype=d)  # noqa: E731
            shapes = dict(y=(rows, n), g=(rows, h), u=(rows, h), f=(rows, m), dx=(rows, n), dwg=(h, n), dwu=(h, n), dwd=(m, h), dh=(rows, n), dw=(n,), l=(rows, h))
            t = {k: pad(*s) for k, s in shapes.items()}
            q, s = pad(rows, n, d=torch.int8), pad(rows, d=torch.float32)
            ops.norm_fw(x, None, w, None, t["y"][:rows * n].view(rows, n))
            ops.norm_int8(x, None, w, None, q, s)
            ops.linear_int8(q[:rows * n].view(rows, n), s, wq, wqs, None, t["l"])
            ops.ffn_fw(x, wg, wu, wd, t["g"], t["u"], t["f"])
            ops.ffn_bw(x, wg, wu, wd, t["g"], t["u"], dy, t["dx"], t["dwg"], t["dwu"], t["dwd"])
            ops.norm_bw(x, w, t["dx"], None, t["dh"], t["dw"])
            for k, shape in shapes.items():
                assert (t[k][int(np.prod(shape)):] == 77).all(), k
            assert (q[rows * n:] == 77).all() and (s[rows:] == 77).all()
            now = [v.clone() for v in t.values()] + [q, s]
            assert first is None or all(torch.equal(a, b) for a, b in zip(first, now))
            first = now


@both
@pytest.mark.parametrize("size", [40, 300, 1001, 4096, 40000])
def test_ties_between_two_steps_go_to_the_even_one(ops, size, dt):
    """values that lie in the middle of two steps: half of a row's largest magnitude (63.5 steps), and in rows whose largest magnitude is 127 times a
    power of two every half step.  Whole numbers: the same ones from the rows, and from the norm with weights of one (its h times 1 is rounded nowhere)."""
    rows = 64
    x = randn(120, rows, size, dt=dt).clamp(-4, 4)
    top = (4 + randn(121, rows).abs()).to(dt)                            # (a half of them is a number of either type, too)
    x[:, 0], x[:, 3], x[:, size - 1] = top, top / 2, -top / 2
    want = torch.round(x.double() * 127 / top.double()[:, None])         # 127 x is exact in 64 bits, and the quotient of a tie a whole number and a half
    assert (want[:, 3] == 64).all() and (want[:, size - 1] == -64).all()
    steps = torch.arange(size, device="cuda") % 254 - 126.5
    power = 2.0 ** (torch.arange(rows, device="cuda") % 9 - 4)
    y = (steps[None, :] * power[:, None]).to(dt)
    y[:, 1] = (127 * power).to(dt)
    even = torch.round(steps.double())[None, :].repeat(rows, 1)
    even[:, 1] = 127
    q, scale, ones = blank(rows, size, dt=torch.int8), blank(rows), torch.ones(size, device="cuda", dtype=dt)
    for shift in (0, 1):
        for v, whole in ((x, want), (y, even)):
            room = blank(rows, size, dt=dt, shift=shift).copy_(v)
            ops.rows_int8(room, q, scale)
            assert torch.equal(q.double(), whole)
            ops.norm_int8(room, None, ones, None, q, scale)
            assert torch.equal(q.double(), whole)


@both
@pytest.mark.parametrize("size", [5, 34, 96, 1000, 1001, 4096, 16384, 40000])
def test_norm_weights_that_are_no_numbers(ops, size, dt):
    """a weight that is NaN or infinite is part of every row: in 8 bits no row has a finite scale, and q is 0 in the NaN's column; also where
    every other value of the row is zero.  The sum that goes on along the residual path keeps its bits."""
    rows = 5
    x, res = randn(130, rows, size, dt=dt), randn(131, rows, size, dt=dt)
    x[1], res[1] = 0, 0
    w = (1 + randn(132, size, scale=0.3)).to(dt)
    clean = blank(rows, size, dt=dt)
    ops.norm_fw(x, res, w, clean, blank(rows, size, dt=dt))
    for shift in (0, 1):
        a, b = blank(rows, size, dt=dt, shift=shift).copy_(x), blank(rows, size, dt=dt, shift=shift).copy_(res)
        for what in (float("nan"), float("inf"), -float("inf")):
            for at in (0, size // 2, size - 1):
                bad = w.clone()
                bad[at] = what
                total, q, scale = blank(rows, size, dt=dt, shift=shift), blank(rows, size, dt=torch.int8, shift=shift), blank(rows)
                ops.norm_int8(a, b, bad, total, q, scale)
                assert not torch.isfinite(scale).any(), (what, at)
                assert (q[:, at] == 0).all(), (what, at)
                assert torch.equal(total, clean)


@pytest.mark.parametrize("h", [16, 40, 258, 1026, 2730, 4096])
@pytest.mark.parametrize("rows", [1, 2, 5, 8])
def test_ffn_few_halves_pass_the_gated_product_on_in_two_parts(ops, rows, h):
    """Up to eight tokens in half precision silu(gate) * up reaches the second product as itself and what its rounding left.  Seen where results cancel:
    columns 2 j and 2 j + 1 have the same gate and ups whose quotient is 1 + 2^-10, and result j is their difference, 2^-10 H.  H rounded once would
    be off by up to half of that; in two parts what counts, relative to H, is: 2^-22 of either column (the second part's rounding), n + 1 roundings
    or cuts of 2^-23 in either up and its product with silu(gate) (the gates are the same bits), and 2^-22 at each of the four terms that the sum adds."""
    dt, n = torch.float16, 8
    m = h // 2
    x = (1 + randn(140, rows, n).abs().clamp(max=1)).to(dt)
    wg = (randn(141, m, n).abs() / n).to(dt).repeat_interleave(2, 0)
    wu = torch.ones(h, n, device="cuda", dtype=dt)
    wu[1::2] = 1 + 2.0 ** -10
    wd = torch.zeros(m, h, device="cuda", dtype=dt)
    at = torch.arange(m, device="cuda")
    wd[at, 2 * at], wd[at, 2 * at + 1] = -1, 1
    gd, ud = x.double() @ wg.double().T, x.double() @ wu.double().T
    hd = silu(gd) * ud
    want, size = hd @ wd.double().T, hd[:, 1::2]
    for shift in (0, 1):
        y = blank(rows, m, dt=dt, shift=shift)
        ops.ffn_fw(*[blank(*t.shape, dt=dt, shift=shift).copy_(t) for t in (x, wg, wu, wd)], None, None, y)
        within(y, want, want.abs() * (HALF[dt] + 2.0 ** -16) + size * (2 * 2.0 ** -22 + 2 * (n + 1) * 2.0 ** -23 + 4 * 2.0 ** -22), "y")


@both
def test_on_the_default_stream(ops, dt):
    """cudaStreamLegacy, where torch's own kernels are queued: behind the one that makes the input and in front of the one that reads the result, without a
    wait on the host; then the library's own stream again"""
    rows, n, h = 90, 256, 384
    x, wg, wu, wd = ffn_tensors(rows, n, h, n, dt)
    w, y, y2, z, z2 = torch.ones(n, device="cuda", dtype=dt), blank(rows, n, dt=dt), blank(rows, n, dt=dt), blank(rows, n, dt=dt), blank(rows, n, dt=dt)
    ops.norm_fw(x, None, w, None, z)
    ops.ffn_fw(z, wg, wu, wd, None, None, y)
    torch.cuda.synchronize()
    assert torch.cuda.current_stream().cuda_stream == 0
    ops.lib.trainlib_set_stream(1)
    try:
        for turn in range(3):
            late = torch.zeros_like(x)
            for _ in range(20):
                late.copy_(x)
            ops.norm_fw(late, None, w, None, z2, sync=False)
            ops.ffn_fw(z2, wg, wu, wd, None, None, y2, sync=False)
            got, norm = y2.clone(), z2.clone()
            y2.zero_(), z2.zero_()
            assert torch.equal(got, y) and torch.equal(norm, z), turn
    finally:
        torch.cuda.synchronize()
        ops.lib.trainlib_set_stream(None)
    ops.pkg.check(ops.lib)


# ------------------------------------------------------------------------------------------------ tensors whose elements' numbers pass 32 bits
def filled(seed, *shape, dt=torch.float16, scale=1.0):
    """seeded values without a copy in single precision"""
    gen = torch.Generator("cuda").manual_seed(seed)
    if dt == torch.int8:
        return torch.randint(-128, 128, shape, device="cuda", generator=gen, dtype=dt)
    t = torch.empty(shape, device="cuda", dtype=dt).normal_(generator=gen)
    return t.mul_(scale) if scale != 1 else t


@pytest.mark.parametrize("rows,size", [(1048581, 2056), (1048581, 2051), (107401, 20008), (107401, 20003)])
def test_norms_beyond_32_bits(ops, rows, size):
    """more than 2^31 elements: rows in front of, at and behind that border, and the weight's gradient over all of them"""
    dt = torch.float16
    x, w = filled(150, rows, size), (1 + randn(151, size, scale=0.3)).to(dt)
    assert x.numel() > 2 ** 31
    at = torch.tensor([0, 2 ** 31 // size - 1, 2 ** 31 // size, 2 ** 31 // size + 1, rows - 2, rows - 1], device="cuda")
    h = x[at].double()
    want, r = norm_ref(h, w.double())
    y, q, scale = torch.empty_like(x), torch.empty(rows, size, dtype=torch.int8, device="cuda"), blank(rows)
    ops.norm_fw(x, None, w, None, y)
    within(y[at], want, want.abs() * (HALF[dt] + (size / 64 + 16) * U) + TINY[dt], "norm")
    for call, v in ((lambda: ops.norm_int8(x, None, w, None, q, scale), want), (lambda: ops.rows_int8(x, q, scale), h)):
        call()
        step = v.abs().amax(1) / 127
        within(scale[at], step, step * (size / 64 + 16) * U, "scale")
        within(q[at], v / step[:, None], 0.5 + 127 * 8 * U, "q")
    del q, scale
    # backward, dy = the norm's result and a fraction of it, the gradient over it.  The sum over the rows of dy h r is the sum of w (h r)^2, about w times
    # `rows`, in the first pass: beyond 65504 and half a step (65520) that is infinite in half precision.
    for fraction in (1, 2.0 ** -10):
        ops.norm_fw(x, None, w, None, y)
        y.mul_(fraction)
        dy, dw = y[at].double(), blank(size, dt=dt)
        want_dw, terms = torch.zeros(size, device="cuda", dtype=torch.float64), torch.zeros(size, device="cuda", dtype=torch.float64)
        for k in range(0, rows, 65536):
            hk = x[k:k + 65536].double()
            p = y[k:k + 65536].double() * hk / ((hk * hk).mean(1, keepdim=True) + EPS).sqrt()
            want_dw += p.sum(0)
            terms += p.abs().sum(0)
        del hk, p
        ops.norm_bw(x, w, y, None, y, dw)
        g = dy * w.double()
        want = r * (g - h * r * r * (g * h).mean(1, keepdim=True))
        parts = r * g.abs() + h.abs() * r ** 3 * (g * h).abs().mean(1, keepdim=True)
        within(y[at], want, want.abs() * HALF[dt] + parts * (size / 64 + 16) * U + TINY[dt], "dx")
        off = terms * (rows / 32 + size / 64 + 128) * U
        over, fits = want_dw.abs() - off >= 65520, want_dw.abs() + off < 65520
        assert torch.isinf(dw[over]).all() and (fits.all() or fraction == 1)
        if fits.any():
            within(dw[fits], want_dw[fits], (want_dw.abs() * HALF[dt] + off + TINY[dt])[fits], "dweight")


@pytest.mark.parametrize("rows", [2, 20, 40])
@pytest.mark.parametrize("n,h", [(8200, 262147), (8193, 262200)])
def test_ffn_weights_beyond_32_bits(ops, rows, n, h):
    """weights of more than 2^31 elements; only the last hidden columns reach the result and the gradients"""
    dt, m, live = torch.float16, 24, 64
    x, wg, wu = randn(152, rows, n, dt=dt), filled(153, h, n, scale=n ** -0.5), filled(154, h, n, scale=n ** -0.5)
    assert wg.numel() > 2 ** 31
    wd = torch.zeros(m, h, device="cuda", dtype=dt)
    wd[:, h - live:] = randn(155, m, live, scale=live ** -0.5)
    gd, ud = x.double() @ wg[h - live:].double().T, x.double() @ wu[h - live:].double().T
    tail = wd[:, h - live:].double()
    y, g, u = blank(rows, m, dt=dt), blank(rows, h, dt=dt), blank(rows, h, dt=dt)
    ops.ffn_fw(x, wg, wu, wd, g, u, y)
    near(g[:, h - live:], gd, dt, 1, (n,), "gate")
    near(u[:, h - live:], ud, dt, 1, (n,), "up")
    near(y, (silu(gd) * ud) @ tail.T, dt, 2, (3 * n, h), "y", (silu(gd) * ud).square() @ tail.square().T)
    dy, dx, dwu, dwd = randn(156, rows, m, dt=dt), blank(rows, n, dt=dt), torch.empty_like(wu), blank(m, h, dt=dt)
    ops.ffn_bw(x, wg, wu, wd, g, u, dy, dx, None, dwu, dwd)
    want, terms = ffn_bw_ref(x, wg[h - live:], wu[h - live:], wd[:, h - live:], g[:, h - live:], u[:, h - live:], dy)
    near(dx, want[0], dt, 2, (m, 2 * h), "dx", terms[0])
    near(dwu[h - live:], want[2], dt, 2, (m, rows), "dw_up", terms[2])
    near(dwd[:, h - live:], want[3], dt, 2, (m, rows), "dw_down", terms[3])
    assert (dwu[:h - live].amax(1) == 0).all() and (dwu[:h - live].amin(1) == 0).all()


@pytest.mark.parametrize("h", [32776, 32771])
def test_ffn_tokens_beyond_32_bits(ops, h):
    """projections of more than 2^31 elements"""
    dt, rows, n, m, live = torch.float16, 65600, 72, 40, 128
    x, wg, wu, wd = ffn_tensors(rows, n, h, m, dt)
    y, g, u = blank(rows, m, dt=dt), torch.empty(rows, h, device="cuda", dtype=dt), torch.empty(rows, h, device="cuda", dtype=dt)
    assert g.numel() > 2 ** 31
    ops.ffn_fw(x, wg, wu, wd, g, u, y)
    gd, ud = x[-live:].double() @ wg.double().T, x[-live:].double() @ wu.double().T
    near(g[-live:], gd, dt, 1, (n,), "gate")
    near(u[-live:], ud, dt, 1, (n,), "up")
    near(y[-live:], (silu(gd) * ud) @ wd.double().T, dt, 2, (3 * n, h), "y", (silu(gd) * ud).square() @ wd.double().square().T)
    del gd, ud
    dy = randn(157, rows, m, dt=dt)
    got = [blank(*t.shape, dt=dt) for t in (x, wg, wu, wd)]
    ops.ffn_bw(x, wg, wu, wd, g, u, dy, *got)
    want, terms = ffn_bw_ref(x[-live:], wg, wu, wd, g[-live:], u[-live:], dy[-live:])
    near(got[0][-live:], want[0], dt, 2, (m, 2 * h), "dx", terms[0])
    want, terms = ffn_bw_ref(x, wg[-live:], wu[-live:], wd[:, -live:], g[:, -live:], u[:, -live:], dy)
    for k, (t, v, q, what) in enumerate(zip(got, want, terms, ("dx", "dw_gate", "dw_up", "dw_down"))):
        if k:
            near(t[:, -live:] if k == 3 else t[-live:], v, dt, 2, (m, rows), what, q)


@pytest.mark.parametrize("rows", [2, 20, 40])
@pytest.mark.parametrize("n", [32016, 32007])
def test_linear_in_8_bits_beyond_32_bits(ops, rows, n):
    m, live = 70001, 40
    x, w = filled(158, rows, n, dt=torch.int8), filled(159, m, n, dt=torch.int8)
    assert w.numel() > 2 ** 31
    y = blank(rows, m)
    ops.linear_int8(x, torch.ones(rows, device="cuda"), w, torch.ones(m, device="cuda"), None, y)
    for cols in (slice(0, live), slice(2 ** 31 // n - live // 2, 2 ** 31 // n + live // 2), slice(m - live, m)):
        assert torch.equal(y[:, cols], (x.double() @ w[cols].double().T).float())


@both
@pytest.mark.parametrize("rows", [6, 70])
def test_alternating_between_streams(ops, rows, dt):
    """two streams of the caller in turn: the scratch that their calls share passes from one to the other, and each result is its own"""
    n, h = 260, 1000
    progs = []
    for k in range(2):
        x, wg, wu, wd = ffn_tensors(rows, n, h, n, dt, seed=160 + 10 * k)
        y, g, u = blank(rows, n, dt=dt), blank(rows, h, dt=dt), blank(rows, h, dt=dt)
        dy, w = randn(165 + 10 * k, rows, n, dt=dt), (1 + randn(166 + 10 * k, n, scale=0.2)).to(dt)
        grads = [blank(*t.shape, dt=dt) for t in (x, wg, wu, wd)] + [blank(rows, n, dt=dt), blank(n, dt=dt)]

        def step(x=x, ws=(wg, wu, wd), y=y, g=g, u=u, dy=dy, w=w, grads=grads):
            ops.ffn_fw(x, *ws, g, u, y, sync=False)
            ops.ffn_bw(x, *ws, g, u, dy, *grads[:4], sync=False)
            ops.norm_bw(y, w, grads[0], dy, grads[4], grads[5], sync=False)
        torch.cuda.synchronize()
        step()
        ops.lib.trainlib_synchronize()
        outs = [y, g, u] + grads
        progs.append((step, outs, [t.clone() for t in outs]))
    streams = [torch.cuda.Stream() for _ in range(2)]
    for turn in range(8):
        for _, outs, _ in progs:
            for t in outs:
                t.fill_(3)
        torch.cuda.synchronize()
        for _ in range(3):
            for s, (step, _, _) in zip(streams, progs):
                ops.lib.trainlib_set_stream(s.cuda_stream)
                step()
        torch.cuda.synchronize()
        for _, outs, first in progs:
            assert all(torch.equal(a, b) for a, b in zip(outs, first)), turn
    ops.lib.trainlib_set_stream(None)
    ops.pkg.check(ops.lib)


@both
@pytest.mark.parametrize("rows,n,h,m", [(7, 72, 200, 40), (65, 130, 257, 63), (300, 264, 520, 136)])
def test_ffn_gradients_in_every_combination(ops, rows, n, h, m, dt):
    """each set of wanted gradients, and nothing written for the others"""
    x, wg, wu, wd = ffn_tensors(rows, n, h, m, dt)
    g, u, dy = randn(170, rows, h, dt=dt), randn(171, rows, h, dt=dt), randn(172, rows, m, dt=dt)
    want, terms = ffn_bw_ref(x, wg, wu, wd, g, u, dy)
    for mask in range(1, 16):
        got = [blank(*t.shape, dt=dt) for t in (x, wg, wu, wd)]
        ops.ffn_bw(x, wg, wu, wd, g, u, dy, *[t if mask >> k & 1 else None for k, t in enumerate(got)])
        for k, (t, v, q, l) in enumerate(zip(got, want, terms, (2 * h, rows, rows, rows))):
            if mask >> k & 1:
                near(t, v, dt, 2, (m, l), (mask, k), q)
            else:
                assert (t == 77).all()
