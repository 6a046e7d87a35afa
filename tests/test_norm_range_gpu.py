"""The layer norm on rows that fp32 sums of squares cannot carry: values past about 1e17, values so small that their squares vanish
(with an eps that does not cover them), infinities and NaN; against the formulas in 64 bits.

Such rows are worked out in 64 bits and rounded once to fp32 and once to the result's type, so the bounds of test_norm_gpu.py hold for
them with room to spare; added here is half a step of a subnormal rstd (2^-150), which a row near the end of the range has.
"""
import pytest
import torch

import hipkittensp_b200 as hk
from tests.test_norm_gpu import DEV, U, _check_backward, _depth, _half_step, _reference

pytestmark = pytest.mark.gpu

# one warp to sixteen per row, three and four chunks per thread, rows off every boundary, rows longer than the registers
WIDTHS = [2, 33, 512, 768, 1001, 1024, 2048, 4096, 5003, 8192, 12288, 16384, 20000, 20001]


def _noise(rows, H, seed):
    g = torch.Generator(device=DEV).manual_seed(seed + H)
    return torch.randn(rows, H, generator=g, device=DEV)


def _parameters(H, dtype):
    p = _noise(2, H, 77)
    return (1 + 0.3 * p[0]).to(dtype), (0.3 * p[1]).to(dtype)


def _check(x, w, b, eps, y, mean, rstd):
    H = x.shape[1]
    rm, _, rr, xhat, ry = _reference(x, w, b, eps)
    dm = (_depth(H) + 3) * U * (x.double() - rm[:, None]).abs().mean(1) + 2 * U * rm.abs() + 1e-38
    rel = 0.5 * ((_depth(H) + 8) * U + dm * dm * rr * rr) + 3 * U
    assert ((mean.double() - rm).abs() <= dm).all()
    assert ((rstd.double() - rr).abs() <= rel * rr + 2.0 ** -150).all()
    xw = (xhat * w.double()).abs()
    tol = w.double().abs() * (rr * dm)[:, None] + xw * (rel + 4 * U)[:, None] + 2 * U * (xw + b.double().abs()) + _half_step(y.dtype) * ry.abs() * 1.01 + 1e-38
    bad = ~((y.double() - ry).abs() <= tol)             # (a NaN is bad)
    assert not bad.any(), f"rows {bad.any(1).nonzero().flatten().tolist()}"


def _check_gradient(x, dy, w, mean, rstd):
    got = hk.layer_norm_backward(dy, x, mean, rstd, w)
    assert all(torch.isfinite(t).all() for t in got)
    _check_backward(dy, x, mean, rstd, w, *got)


def _large(H, dtype):
    """Ordinary rows between rows of 1e17 to 1e37, with and without a mean, and rows that alternate between both ends of the range."""
    x = _noise(16, H, 5)
    for i, s in enumerate((1e17, 3e17, 1e18, 1e19, 1e30, 1e37)):
        x[2 * i + 1] *= s
    x[3] += 1e18
    x[9] -= 3e30
    x[11] += 2e37
    x[13] = 3e38 * torch.sign(x[13])
    x[15] = 1e37 * torch.sign(x[15]).abs()
    return x.to(dtype)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("H", WIDTHS)
def test_large_rows(H, dtype):
    x = _large(H, dtype)
    w, b = _parameters(H, dtype)
    y, mean, rstd = hk.layer_norm(x, w, b)
    _check(x, w, b, 1e-5, y, mean, rstd)
    # a constant row has variance 0, whatever its size
    assert torch.equal(y[15], b) and torch.equal(mean[15], x[15, 0].float()) and abs(rstd[15].item() * 1e-5 ** 0.5 - 1) <= 4 * U
    # the rows beside them keep their bits
    plain = x.clone()
    plain[1::2] = 0
    for got, want in zip((y, mean, rstd), hk.layer_norm(plain, w, b)):
        assert torch.equal(got[::2], want[::2])
    z = x.clone()
    assert torch.equal(hk.layer_norm(z, w, b, out=z)[0], y)
    # rows that lie apart from their result, element by element
    apart = torch.empty(x.numel() + 1, dtype=dtype, device=DEV)[1:].view(x.shape)
    apart.copy_(x)
    _check(x, w, b, 1e-5, *hk.layer_norm(apart, w, b))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("H", [512, 1001, 4096, 12000, 20000])
def test_gradient_of_large_rows(H, dtype):
    x, dy = _large(H, dtype)[:13], _noise(13, H, 9).to(dtype)
    w, b = _parameters(H, dtype)
    _, mean, rstd = hk.layer_norm(x, w, b)
    _check_gradient(x, dy, w, mean, rstd)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("H", WIDTHS[1:])
def test_small_rows_without_eps(H, dtype):
    x = _noise(12, H, 6)
    for i, s in enumerate((1e-10, 1e-17, 1e-22, 1e-30, 1e-35)):
        x[2 * i + 1] *= s
    x = x.to(dtype)
    w, b = _parameters(H, dtype)
    for eps in (0.0, 1e-30):
        _check(x, w, b, eps, *hk.layer_norm(x, w, b, eps=eps))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("H", WIDTHS)
def test_statistics_of_rows_with_infinities_and_nan(H, dtype):
    """mean is the sum over H (infinite, or NaN where infinities meet), rstd and the row are NaN; the rows beside keep their bits."""
    inf, nan = float("inf"), float("nan")
    x = _noise(11, H, 7).to(dtype)
    w, b = _parameters(H, dtype)
    ref = hk.layer_norm(x, w, b)
    x[1, 0] = inf
    x[3, H - 1] = -inf
    x[5, H // 2] = nan
    x[7, 0], x[7, H - 1] = inf, -inf
    x[9] = -inf
    y, mean, rstd = hk.layer_norm(x, w, b)
    assert mean[1] == inf and mean[3] == -inf and mean[9] == -inf and torch.isnan(mean[[5, 7]]).all()
    assert torch.isnan(rstd[1::2]).all() and torch.isnan(y[1::2]).all()
    for got, want in zip((y, mean, rstd), ref):
        assert torch.equal(got[::2], want[::2])


@pytest.mark.parametrize("fmt", [hk.E2M3, hk.E3M2, hk.E4M3, hk.E5M2, hk.E2M1])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("H", [32, 512, 1056, 4096, 8192, 16384, 20000])
def test_large_rows_to_operand(H, dtype, fmt):
    """The bits of the plain norm followed by the quantiser, for large rows, infinities and NaN too."""
    x = _large(H, dtype)
    x[4, 3], x[6, 5] = float("inf"), float("nan")
    w, b = (t.float() for t in _parameters(H, dtype))
    packed, scales, mean, rstd = hk.layer_norm_quantize(x, w, b, fmt=fmt)
    y, m, r = hk.layer_norm(x.float(), w, b)
    wp, ws = hk.quantize(y, fmt)
    assert torch.equal(packed, wp) and torch.equal(scales, ws)
    good = [i for i in range(16) if i not in (4, 6)]
    assert torch.equal(mean[good], m[good]) and torch.equal(rstd[good], r[good])
    assert torch.isnan(rstd[[4, 6]]).all()


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("H", [512, 768, 1001, 20000])
def test_gradient_sums_that_overflow_stay_infinite(H, dtype):
    """sum(g) past the range of fp32 is an infinity, as a plain fp32 sum of such terms is, not a NaN: dx = (g - inf - 0) * rstd = -inf."""
    x = torch.zeros(3, H, dtype=dtype, device=DEV)
    dy = torch.zeros_like(x)
    dy[1] = 3e38
    mean, rstd = torch.zeros(3, device=DEV), torch.ones(3, device=DEV)
    dx = hk.layer_norm_backward(dy, x, mean, rstd)[0]
    assert torch.isneginf(dx[1]).all() and not dx[[0, 2]].any()


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("H", [33, 256, 700, 1001, 4001, 8190, 9001, 16001, 20001])
def test_gradient_of_constant_rows_far_from_zero(H, dtype):
    """Rows of one large value: xhat is 0 and rstd 1 / sqrt(eps), and a mean that is an infinite number of rstd from 0 reaches no element."""
    x = torch.full((9, H), 2e36, dtype=dtype, device=DEV)
    x[::2] = _noise(5, H, 3).to(dtype)
    dy = _noise(9, H, 4).to(dtype)
    w, b = _parameters(H, dtype)
    _, mean, rstd = hk.layer_norm(x, w, b)
    _check_gradient(x, dy, w, mean, rstd)


def test_results_that_share_bytes_are_refused():
    x, dy = _noise(8, 64, 1), _noise(8, 64, 2)
    w, b = _parameters(64, torch.float32)
    flat = torch.zeros(8 * 64 + 64, device=DEV)
    flat[512:] = w
    with pytest.raises(RuntimeError, match="overlaps weight"):
        hk.layer_norm(x, flat[512:], b, out=flat[8:520].view(8, 64))
    hk.layer_norm(x, flat[512:], b, out=flat[:512].view(8, 64))                       # neighbours
    assert torch.equal(flat[512:], w) and torch.equal(flat[:512].view(8, 64), hk.layer_norm(x, w, b)[0])
    _, mean, rstd = hk.layer_norm(x, w, b)
    need = hk.lib.mxfp6_layer_norm_backward_workspace_bytes(8, 64)
    buf = torch.zeros(need + 4096, dtype=torch.uint8, device=DEV)
    dx, sums, st = torch.empty_like(x), torch.empty(128, device=DEV), torch.cuda.current_stream().cuda_stream

    def call(dw, db, ws):
        return hk.lib.mxfp6_layer_norm_backward(dy.data_ptr(), x.data_ptr(), 0, mean.data_ptr(), rstd.data_ptr(), w.data_ptr(), 0, dx.data_ptr(), dw, db, 8, 64, ws, need, st)

    s, p = sums.data_ptr(), buf.data_ptr()
    assert call(s, s + 256, p) == 0
    for bad in ((s, s, p), (s, s + 252, p), (dx.data_ptr(), s, p), (s, dx.data_ptr() + 2044, p), (p, s, p), (s, p + need - 4, p)):
        assert call(*bad) == 1 and b"overlaps" in hk.lib.mxfp6_last_error(), bad
    for t in (dx, x, dy, w, mean, rstd):
        assert call(s, s + 256, t.data_ptr()) == 1 and b"overlaps" in hk.lib.mxfp6_last_error()
