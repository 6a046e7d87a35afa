"""Layer norm, its MX form and its gradient on the GPU against the formulas in 64 bits.

Tolerances, to first order in u = 2^-24 (half a step of fp32) and ut (half a step of the result's type).  A kernel sum of H terms
is a chain of at most `depth` additions per term, so its error is at most depth * u * sum|terms|.

  mean       the second pass sums the distances from the first mean, so what is left is the rounding of the mean itself and of the
             distances: (depth + 3) u mean|x - mean| + 2u |mean|                                                       =: dm
  rstd       the variance is a sum of positive terms, each (1 + 4u): relative (depth + 8) u, plus (dm / std)^2; rstd half of it, plus 3u
  y          |w| rstd dm + |xhat w| (relative error of rstd + 4u) + 2u (|xhat w| + |b|) + ut |y|
  dx         g and xhat carry 4u each; the row sums depth * u * sum|terms|
  dw, db     a chain of the rows of one CTA, its share of the partials and five pairwise steps
"""
import numpy as np
import pytest
import torch

import hipkittensp_b200 as hk
from oracle import mxfp6_ref as R

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
DEV = "cuda"


def _depth(H):
    return 32 * max(1, -(-H // 16384)) + 10


def _inputs(rows, H, dtype, wdtype=None, seed=0, spread=True):
    g = torch.Generator(device=DEV).manual_seed(seed + rows * 7 + H)
    n = lambda *s: torch.randn(*s, generator=g, device=DEV)
    x = n(rows, H)
    if spread:
        x = x * torch.exp(n(rows, 1)) + 3 * n(rows, 1)
    wd = dtype if wdtype is None else wdtype
    return x.to(dtype), (1 + 0.3 * n(H)).to(wd), (0.3 * n(H)).to(wd), n(rows, H).to(dtype)


def _reference(x, w, b, eps):
    x, w, b = x.double(), w.double(), b.double()
    mean = x.mean(1)
    d = x - mean[:, None]
    var = (d * d).mean(1)
    rstd = 1 / torch.sqrt(var + eps)
    xhat = d * rstd[:, None]
    return mean, var, rstd, xhat, xhat * w + b


def _half_step(t):
    return torch.finfo(t).eps / 2


def _check_forward(x, w, b, eps, y, mean, rstd):
    H = x.shape[1]
    rm, rv, rr, xhat, ry = _reference(x, w, b, eps)
    d = (x.double() - rm[:, None]).abs()
    dm = (_depth(H) + 3) * U * d.mean(1) + 2 * U * rm.abs() + 1e-38
    rel = 0.5 * ((_depth(H) + 8) * U + dm * dm * rr * rr) + 3 * U
    assert ((mean.double() - rm).abs() <= dm).all()
    assert ((rstd.double() - rr).abs() <= rel * rr).all()
    if y is None:
        return
    xw = (xhat * w.double()).abs()
    tol = w.double().abs() * (rr * dm)[:, None] + xw * (rel + 4 * U)[:, None] + 2 * U * (xw + b.double().abs()) + _half_step(y.dtype) * ry.abs() * 1.01 + 1e-38
    bad = (y.double() - ry).abs() > tol
    assert not bad.any(), f"{int(bad.sum())} of {bad.numel()} elements, worst {((y.double() - ry).abs() / tol).max().item():.2f} of the bound"


WIDTHS = [1, 2, 3, 7, 8, 9, 31, 32, 96, 249, 250, 255, 256, 264, 505, 506, 512, 520, 1001, 1017, 1018, 1024, 1032, 2041, 2042, 2048, 2056, 4090, 4095, 4096, 5000, 8185, 8186,
          8192, 8200, 16377, 16378, 16384, 16392, 16385, 40000]


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("H", WIDTHS)
def test_forward(H, dtype):
    rows = 700 if H <= 2048 else 37
    x, w, b, _ = _inputs(rows, H, dtype)
    y, mean, rstd = hk.layer_norm(x, w, b)
    _check_forward(x, w, b, 1e-5, y, mean, rstd)


@pytest.mark.parametrize("rows", [0, 1, 2, 7, 8, 9, 149, 5000])
@pytest.mark.parametrize("H", [64, 1000, 4096])
def test_forward_row_counts(rows, H):
    x, w, b, _ = _inputs(rows, H, torch.bfloat16, torch.float32)
    y, mean, rstd = hk.layer_norm(x, w, b, eps=1e-6)
    assert y.shape == x.shape and mean.shape == (rows,)
    if rows:
        _check_forward(x, w, b, 1e-6, y, mean, rstd)


def test_forward_without_parameters_in_place_and_unaligned():
    x, w, b, _ = _inputs(33, 768, torch.bfloat16)
    one, zero = torch.ones_like(w), torch.zeros_like(w)
    assert torch.equal(hk.layer_norm(x)[0], hk.layer_norm(x, one, zero)[0])
    assert torch.equal(hk.layer_norm(x, w)[0], hk.layer_norm(x, w, zero)[0])
    assert torch.equal(hk.layer_norm(x, None, b)[0], hk.layer_norm(x, one, b)[0])
    want = hk.layer_norm(x, w, b)[0]
    z = x.clone()
    assert hk.layer_norm(z, w, b, out=z)[0].data_ptr() == z.data_ptr() and torch.equal(z, want)
    # rows that start one element off every vector boundary, inside a buffer whose other elements stay as they were
    buf = torch.full((33 * 768 + 2,), 7.0, dtype=torch.bfloat16, device=DEV)
    xs, ys = torch.empty(33 * 768 + 1, dtype=torch.bfloat16, device=DEV)[1:].view(33, 768), buf[1:-1].view(33, 768)
    xs.copy_(x)
    y, mean, rstd = hk.layer_norm(xs, w, b, out=ys)
    _check_forward(x, w, b, 1e-5, y, mean, rstd)
    assert buf[0] == 7 and buf[-1] == 7


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("rows,H", [(1, 5), (40, 9), (500, 33), (777, 1003), (300, 3001), (5000, 67), (200, 16370)])
@pytest.mark.parametrize("start", [0, 1, 5])
def test_rows_that_start_anywhere(rows, H, dtype, start):
    """Rows of odd widths from a buffer that starts off every vector boundary: nothing beside the rows is written, and what lies
    there (NaN) is not read; both passes, many rows per CTA and few."""
    x, w, b, dy = _inputs(rows, H, dtype)
    n = rows * H
    make = lambda t: torch.full((n + 16,), float("nan"), dtype=dtype, device=DEV)
    bufs = [make(t) for t in range(4)]
    xs, ys, gs, ds = (t[start:start + n].view(rows, H) for t in bufs)
    xs.copy_(x)
    gs.copy_(dy)
    y, mean, rstd = hk.layer_norm(xs, w, b, out=ys)
    _check_forward(x, w, b, 1e-5, y, mean, rstd)
    dw, db = torch.empty(H, device=DEV), torch.empty(H, device=DEV)
    nbytes = hk.lib.mxfp6_layer_norm_backward_workspace_bytes(rows, H)
    work = torch.empty(nbytes, dtype=torch.uint8, device=DEV)
    for dx in (ds, torch.empty(n + 16, dtype=dtype, device=DEV)[(start + 1) % 8:][:n].view(rows, H)):      # the second lies apart from x and dy
        rc = hk.lib.mxfp6_layer_norm_backward(gs.data_ptr(), xs.data_ptr(), 0 if dtype == torch.float32 else 1, mean.data_ptr(), rstd.data_ptr(), w.data_ptr(),
                                              0 if dtype == torch.float32 else 1, dx.data_ptr(), dw.data_ptr(), db.data_ptr(), rows, H, work.data_ptr(), nbytes,
                                              torch.cuda.current_stream().cuda_stream)
        assert rc == 0, hk.lib.mxfp6_last_error()
        _check_backward(dy, x, mean, rstd, w, dx, dw, db)
    for t in bufs:
        assert torch.isnan(t[:start]).all() and torch.isnan(t[start + n:]).all()


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_forward_far_mean_constant_rows_and_bad_values(dtype):
    """Rows whose mean is 10^4 times their spread keep their digits (E[x^2] - mean^2 would lose them all); a constant row has
    variance 0; an infinity or a NaN stays in its own row."""
    H = 4096
    x, w, b, _ = _inputs(12, H, torch.float32, spread=False)
    x[1] += 1e4
    x[2] = 3.25
    x[3] = 0.0
    x[4] *= 1e-20
    x[5] *= 1e15
    x = x.to(dtype)
    _check_forward(x, w, b, 1e-5, *hk.layer_norm(x, w, b))
    good = [0, 1, 2, 3, 4, 5, 6, 8, 10, 11]
    ref = hk.layer_norm(x, w, b)
    x[7, 100] = float("inf")
    x[9, 4000] = float("nan")
    y, mean, rstd = hk.layer_norm(x, w, b)
    assert torch.isnan(y[[7, 9]]).all()
    for got, want in zip((y, mean, rstd), ref):
        assert torch.equal(got[good], want[good])


def _codes_match(x, w, b, fmt, packed, scales):
    """Codes against the quantised 64-bit result: another scale only where the largest value lies at a power of two, another code
    only where a value lies at a rounding boundary, and never further than one step of the block."""
    ry = _reference(x, w, b, 1e-5)[4]
    wp, ws = R.quantize(ry.float().cpu().numpy(), fmt)
    gp, gs = packed.cpu().numpy(), scales.cpu().numpy()
    assert np.abs(gs.astype(int) - ws).max() <= 1
    assert (gs != ws).mean() <= 1e-3
    same = (gs == ws).repeat(32, axis=1)
    assert (R.codes_of(gp, fmt) != R.codes_of(wp, fmt))[same].mean() <= 1e-3
    p = R._FMT[fmt]
    step = np.ldexp(1.0, np.maximum(gs, ws).astype(int) - 127 + p["emax"] - p["mbits"]).repeat(32, axis=1)
    assert (np.abs(R.dequantize(gp, gs, fmt) - R.dequantize(wp, ws, fmt)) <= step).all()


@pytest.mark.parametrize("fmt", [R.E2M3, R.E3M2, R.E4M3, R.E5M2, R.E2M1])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("H", [32, 96, 256, 480, 1024, 1056, 2048, 4096, 8192, 16384, 20000])
def test_forward_to_operand(H, dtype, fmt):
    rows = 300 if H <= 1056 else 21
    x, w, b, _ = _inputs(rows, H, dtype, torch.float32)
    packed, scales, mean, rstd = hk.layer_norm_quantize(x, w, b, fmt=fmt)
    _check_forward(x, w, b, 1e-5, None, mean, rstd)
    _codes_match(x, w, b, fmt, packed, scales)
    # the same arithmetic as the plain norm of the same values followed by the quantiser, bit for bit
    y = hk.layer_norm(x.float(), w, b)[0]
    wp, ws = hk.quantize(y, fmt)
    assert torch.equal(packed, wp) and torch.equal(scales, ws)


@pytest.mark.parametrize("fmt", [R.E2M3, R.E4M3, R.E2M1])
def test_norm_into_product(fmt):
    """Norm, operand and 4-bit product together, against the 64-bit product of what the operand holds; then the norm's gradient
    for the gradient of that product, against automatic differentiation in 64 bits."""
    rows, H, N = 200, 1024, 640
    x, w, b, _ = _inputs(rows, H, torch.bfloat16, torch.float32, seed=5)
    weight = torch.randn(N, H, generator=torch.Generator(device=DEV).manual_seed(9), device=DEV) * 0.05
    wp, ws = hk.quantize(weight, hk.E2M1)
    packed, scales, mean, rstd = hk.layer_norm_quantize(x, w, b, fmt=fmt)
    c = hk.gemm(packed, scales, wp, ws, fmt=fmt, fmt_b=hk.E2M1)
    assert hk.device_status() == 0
    A, B = hk.dequantize(packed, scales, fmt).double(), hk.dequantize(wp, ws, hk.E2M1).double()
    # fp32 accumulation of H terms (at most H u sum|terms|) and one rounding to bf16
    tol = _half_step(torch.bfloat16) * (A @ B.t()).abs() * 1.01 + H * U * (A.abs() @ B.abs().t())
    assert ((c.double() - A @ B.t()).abs() <= tol).all()
    dc = torch.randn(rows, N, generator=torch.Generator(device=DEV).manual_seed(3), device=DEV)
    dy = (dc @ B.float()).to(torch.bfloat16)
    _check_backward(dy, x, mean, rstd, w, *hk.layer_norm_backward(dy, x, mean, rstd, w))
    leaf = [t.double().requires_grad_() for t in (x, w, b)]
    y = torch.nn.functional.layer_norm(leaf[0], (H,), leaf[1], leaf[2], 1e-5)
    grads = torch.autograd.grad((y * dy.double()).sum(), leaf)
    for got, want in zip(hk.layer_norm_backward(dy, x, mean, rstd, w), grads):
        assert (got.double() - want).norm() <= 4e-3 * want.norm()      # dx is rounded to bf16 (at most 2^-8 of each element)


# ---------------------------------------------------------------------------------- backward
def _check_backward(dy, x, mean, rstd, w, dx, dw, db):
    rows, H = x.shape
    dy, x, wt = dy.double(), x.double(), torch.ones(H, dtype=torch.float64, device=DEV) if w is None else w.double()
    m, r = mean.double()[:, None], rstd.double()[:, None]
    xhat, g = (x - m) * r, dy * wt
    m1, m2 = g.mean(1, keepdim=True), (g * xhat).mean(1, keepdim=True)
    ref = (g - m1 - xhat * m2) * r
    d = _depth(H) if H <= 16384 else H // 1024 + 12
    e1 = (d + 4) * U * g.abs().mean(1, keepdim=True)
    e2 = (d + 8) * U * (g * xhat).abs().mean(1, keepdim=True)
    tol = r * (e1 + xhat.abs() * e2 + 6 * U * (g.abs() + m1.abs() + 2 * (xhat * m2).abs())) + _half_step(dx.dtype) * ref.abs() * 1.01 + 1e-38
    bad = (dx.double() - ref).abs() > tol
    assert not bad.any(), f"{int(bad.sum())} of {bad.numel()} elements of dx"
    parts = max(1, hk.lib.mxfp6_layer_norm_backward_workspace_bytes(rows, H) // (8 * (H + 14)))
    chain = -(-rows // parts) + -(-parts // 32) + 16
    assert ((dw.double() - (dy * xhat).sum(0)).abs() <= (chain + 6) * U * (dy * xhat).abs().sum(0) + 1e-38).all()
    assert ((db.double() - dy.sum(0)).abs() <= (chain + 2) * U * dy.abs().sum(0) + 1e-38).all()


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("H", WIDTHS)
def test_backward(H, dtype):
    rows = 900 if H <= 2048 else 200
    x, w, b, dy = _inputs(rows, H, dtype)
    _, mean, rstd = hk.layer_norm(x, w, b)
    got = hk.layer_norm_backward(dy, x, mean, rstd, w)
    assert got[0].dtype == dtype and got[1].dtype == got[2].dtype == torch.float32
    _check_backward(dy, x, mean, rstd, w, *got)
    again = hk.layer_norm_backward(dy, x, mean, rstd, w)
    assert all(torch.equal(a, c) for a, c in zip(got, again))


@pytest.mark.parametrize("rows", [1, 2, 9, 150, 3000])
@pytest.mark.parametrize("H", [64, 1000, 4096, 8193])
def test_backward_row_counts(rows, H):
    x, w, b, dy = _inputs(rows, H, torch.bfloat16, torch.float32)
    _, mean, rstd = hk.layer_norm(x, w, b)
    _check_backward(dy, x, mean, rstd, w, *hk.layer_norm_backward(dy, x, mean, rstd, w))
    _check_backward(dy, x, mean, rstd, None, *hk.layer_norm_backward(dy, x, mean, rstd))


def test_backward_of_no_rows_and_unaligned_rows():
    x, w, b, dy = _inputs(0, 96, torch.float32)
    dx, dw, db = hk.layer_norm_backward(dy, x, x.new_empty(0), x.new_empty(0), w)
    assert dx.shape == (0, 96) and not dw.any() and not db.any()
    x, w, b, dy = _inputs(40, 512, torch.bfloat16)
    _, mean, rstd = hk.layer_norm(x, w, b)
    ys = torch.empty(40 * 512 + 1, dtype=torch.bfloat16, device=DEV)[1:].view(40, 512)
    ys.copy_(dy)
    _check_backward(dy, x, mean, rstd, w, *hk.layer_norm_backward(ys, x, mean, rstd, w))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("rows,H", [(70, 512), (70, 1003), (40, 9000), (40, 9001), (20, 20000)])
def test_backward_in_place(rows, H, dtype):
    """dx may be dy or x: the same bits as with a buffer of its own."""
    x, w, b, dy = _inputs(rows, H, dtype)
    _, mean, rstd = hk.layer_norm(x, w, b)
    want = hk.layer_norm_backward(dy, x, mean, rstd, w)
    code = 0 if dtype == torch.float32 else 1
    nbytes = hk.lib.mxfp6_layer_norm_backward_workspace_bytes(rows, H)
    for which in (0, 1):
        xs, gs = x.clone(), dy.clone()
        dx = (gs, xs)[which]
        dw, db, work = torch.empty(H, device=DEV), torch.empty(H, device=DEV), torch.empty(nbytes, dtype=torch.uint8, device=DEV)
        rc = hk.lib.mxfp6_layer_norm_backward(gs.data_ptr(), xs.data_ptr(), code, mean.data_ptr(), rstd.data_ptr(), w.data_ptr(), code, dx.data_ptr(),
                                              dw.data_ptr(), db.data_ptr(), rows, H, work.data_ptr(), nbytes, torch.cuda.current_stream().cuda_stream)
        assert rc == 0, hk.lib.mxfp6_last_error()
        for got, ref in zip((dx, dw, db), want):
            assert torch.equal(got, ref)
        # without the sums no workspace is asked for
        rc = hk.lib.mxfp6_layer_norm_backward(dy.data_ptr(), x.data_ptr(), code, mean.data_ptr(), rstd.data_ptr(), w.data_ptr(), code, dx.data_ptr(),
                                              None, None, rows, H, None, 0, torch.cuda.current_stream().cuda_stream)
        assert rc == 0 and torch.equal(dx, want[0])


@pytest.mark.parametrize("H", [768, 1001])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("wdtype", [torch.float32, torch.bfloat16])
def test_parameter_types_and_optional_statistics(H, dtype, wdtype):
    x, w, b, dy = _inputs(50, H, dtype, wdtype)
    y, mean, rstd = hk.layer_norm(x, w, b)
    _check_forward(x, w, b, 1e-5, y, mean, rstd)
    _check_backward(dy, x, mean, rstd, w, *hk.layer_norm_backward(dy, x, mean, rstd, w))
    code = {torch.float32: 0, torch.bfloat16: 1}
    z, stat, st = torch.empty_like(x), torch.full((50,), 7.0, device=DEV), torch.cuda.current_stream().cuda_stream
    for m, r in ((None, None), (stat.data_ptr(), None), (None, stat.data_ptr())):
        rc = hk.lib.mxfp6_layer_norm(x.data_ptr(), code[dtype], w.data_ptr(), b.data_ptr(), code[wdtype], z.data_ptr(), m, r, 50, H, 1e-5, st)
        assert rc == 0 and torch.equal(z, y)
        assert m is None or torch.equal(stat, mean)
        assert r is None or torch.equal(stat, rstd)
    # one of the two sums alone
    dw, db = hk.layer_norm_backward(dy, x, mean, rstd, w)[1:]
    nbytes = hk.lib.mxfp6_layer_norm_backward_workspace_bytes(50, H)
    work, out = torch.empty(nbytes, dtype=torch.uint8, device=DEV), torch.empty(H, device=DEV)
    for a, c, want in ((out.data_ptr(), None, dw), (None, out.data_ptr(), db)):
        rc = hk.lib.mxfp6_layer_norm_backward(dy.data_ptr(), x.data_ptr(), code[dtype], mean.data_ptr(), rstd.data_ptr(), w.data_ptr(), code[wdtype], z.data_ptr(),
                                              a, c, 50, H, work.data_ptr(), nbytes, st)
        assert rc == 0 and torch.equal(out, want)


@pytest.mark.parametrize("H", [8192, 8191])
def test_matrices_past_32_bits(H):
    """More than 2^31 elements (and 2^32 bytes): the last rows get the bits of a small matrix of the same rows."""
    rows, n = 270000, 64
    x = torch.zeros(rows, H, dtype=torch.bfloat16, device=DEV)
    tail, w, b, dtail = _inputs(n, H, torch.bfloat16, torch.float32)
    x[-n:] = tail
    y, mean, rstd = hk.layer_norm(x, w, b)
    want = hk.layer_norm(tail, w, b)
    assert torch.equal(y[-n:], want[0]) and torch.equal(mean[-n:], want[1]) and torch.equal(rstd[-n:], want[2])
    assert torch.equal(y[0], b.to(torch.bfloat16)) and torch.equal(y[rows // 2], b.to(torch.bfloat16))
    dy = y.zero_()
    dy[-n:] = dtail
    dx, dw, db = hk.layer_norm_backward(dy, x, mean, rstd, w)
    small = hk.layer_norm_backward(dtail, tail, *want[1:], w)
    assert torch.equal(dx[-n:], small[0]) and not dx[:-n].any()
    for got, ref in zip((dw, db), small[1:]):          # the same terms in another order (64 of them are not zero)
        assert ((got - ref).abs() <= 2 * n * U * ref.abs().max()).all()
    del dy, dx, y
    if H % 32 == 0:
        packed, scales, _, _ = hk.layer_norm_quantize(x, w, b, fmt=hk.E2M1)
        sp, ss, _, _ = hk.layer_norm_quantize(tail, w, b, fmt=hk.E2M1)
        assert torch.equal(packed[-n:], sp) and torch.equal(scales[-n:], ss)
        q, qs = hk.quantize(x, hk.E2M1)
        tq, tqs = hk.quantize(tail, hk.E2M1)
        assert torch.equal(q[-n:], tq) and torch.equal(qs[-n:], tqs) and not q[:-n].any()
        d = hk.dequantize(q, qs, hk.E2M1, dtype=torch.bfloat16)
        assert torch.equal(d[-n:], hk.dequantize(tq, tqs, hk.E2M1, dtype=torch.bfloat16)) and not d[:-n].any()


def test_backward_against_differences():
    """d/dx, d/dw and d/db of sum(dy * y) by central differences of the 64-bit formula, at a few places."""
    rows, H, eps = 5, 40, 1e-5
    x, w, b, dy = _inputs(rows, H, torch.float32, spread=False)
    _, mean, rstd = hk.layer_norm(x, w, b, eps=eps)
    dx, dw, db = hk.layer_norm_backward(dy, x, mean, rstd, w)
    f = lambda x, w, b: (dy.double() * _reference(x, w, b, eps)[4]).sum().item()
    h = 1e-4
    for (r, c) in ((0, 0), (2, 17), (4, 39)):
        for leaf, got in ((0, dx[r, c]), (1, dw[c]), (2, db[c])):
            lo, hi = ([t.double().clone() for t in (x, w, b)] for _ in range(2))
            at = (r, c) if leaf == 0 else (c,)
            lo[leaf][at] -= h
            hi[leaf][at] += h
            # the difference quotient is off by h^2 / 6 of the third derivative (of order 10 here) and 1e-16 / h
            assert abs((f(*hi) - f(*lo)) / (2 * h) - got.item()) <= 1e-5 * max(1.0, abs(got.item()))


def test_captured_and_on_other_streams():
    """The operators in one CUDA graph, replayed on new inputs, and on two streams at once."""
    rows, H, N = 64, 1024, 512
    x, w, b, dy = _inputs(rows, H, torch.bfloat16, torch.float32, seed=1)
    wp, ws = hk.quantize(torch.randn(N, H, device=DEV) * 0.05, hk.E2M1)

    def step():
        packed, scales, mean, rstd = hk.layer_norm_quantize(x, w, b, fmt=hk.E2M1)
        return (hk.gemm(packed, scales, wp, ws, fmt=hk.E2M1), hk.dequantize(packed, scales, hk.E2M1), *hk.layer_norm_backward(dy, x, mean, rstd, w),
                *hk.layer_norm(x, w, b))

    step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    for seed in (2, 3):
        nx, _, _, ndy = _inputs(rows, H, torch.bfloat16, torch.float32, seed=seed)
        x.copy_(nx)
        dy.copy_(ndy)
        graph.replay()
        torch.cuda.synchronize()
        for got, want in zip(out, step()):
            assert torch.equal(got, want)
    want = step()
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    results = []
    for _ in range(3):
        for s in streams:
            with torch.cuda.stream(s):
                results.append(hk.layer_norm_backward(dy, x, *hk.layer_norm(x, w, b)[1:], w))
    torch.cuda.synchronize()
    for r in results:
        assert all(torch.equal(a, c) for a, c in zip(r, want[2:5]))
    assert hk.device_status() == 0


def test_refusals():
    x, w, b, dy = _inputs(8, 64, torch.bfloat16)
    _, mean, rstd = hk.layer_norm(x, w, b)
    bad = [lambda: hk.layer_norm(x[:, :32]), lambda: hk.layer_norm(x.half()), lambda: hk.layer_norm(x.view(2, 4, 64)), lambda: hk.layer_norm(x, w[:32]),
           lambda: hk.layer_norm(x, w, b.float()), lambda: hk.layer_norm(x, w.cpu(), b), lambda: hk.layer_norm(x, w.half()), lambda: hk.layer_norm(x, out=x.float()),
           lambda: hk.layer_norm(x, w, b, eps=-1.0), lambda: hk.layer_norm(x[:, :0].contiguous()), lambda: hk.layer_norm_quantize(x[:, :48].contiguous()),
           lambda: hk.layer_norm_quantize(x, fmt=9), lambda: hk.layer_norm_backward(dy.float(), x, mean, rstd), lambda: hk.layer_norm_backward(dy[:4], x, mean, rstd),
           lambda: hk.layer_norm_backward(dy, x, mean[:4], rstd), lambda: hk.layer_norm_backward(dy, x, mean, rstd.double()),
           lambda: hk.layer_norm_backward(dy, x, mean, None), lambda: hk.layer_norm_backward(dy, x, mean, rstd, w[:8])]
    for i, f in enumerate(bad):
        with pytest.raises(RuntimeError):
            f()
            pytest.fail(f"call {i} was not refused")
    # a workspace that is too small, or missing, is refused before anything is launched
    out = torch.zeros(64, device=DEV)
    assert hk.lib.mxfp6_layer_norm_backward(dy.data_ptr(), x.data_ptr(), 1, mean.data_ptr(), rstd.data_ptr(), w.data_ptr(), 1, x.data_ptr(), out.data_ptr(),
                                            out.data_ptr(), 8, 64, None, 0, None) == 1
    assert b"workspace too small" in hk.lib.mxfp6_last_error()
