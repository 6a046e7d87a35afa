"""Layer norm: results that lie on a parameter, a statistic or another result are refused before a device is touched (addresses only)."""
import pytest

import hipkittensp_b200 as hk
from hipkittensp_b200 import _lib

ROWS, H = 5, 64
X, Y, W, B, M, R, S = ((i + 1) << 24 for i in range(7))         # far apart


def _refused(rc):
    return rc == _lib.ERR_BAD_ARG and b"overlaps" in hk.lib.mxfp6_last_error()


@pytest.mark.parametrize("xd,xs", [(0, 4), (1, 2)])
@pytest.mark.parametrize("wd,wsz", [(0, 4), (1, 2)])
def test_forward(xd, xs, wd, wsz):
    def call(y=Y, w=W, b=B, m=M, r=R):
        return hk.lib.mxfp6_layer_norm(X, xd, w, b, wd, y, m, r, ROWS, H, 1e-5, None)

    span, par, st = ROWS * H * xs, H * wsz, ROWS * 4
    for at, size in ((W, par), (B, par), (M, st), (R, st)):
        for y in (at, at - span + xs, at + size - xs):
            assert _refused(call(y=y)), (at, y)
    for at, size in ((X, span), (W, par), (B, par)):
        for m in (at, at - st + 4, at + size - 4):
            assert _refused(call(m=m)) and _refused(call(r=m))
    assert _refused(call(m=R)) and _refused(call(m=R - st + 4))
    # neighbours that only touch are no overlap (there is no device here: the call gets as far as asking for one, or runs on nothing)
    for kw in (dict(rows=0),):
        assert hk.lib.mxfp6_layer_norm(X, xd, W, B, wd, W, W, W, 0, H, 1e-5, None) == _lib.OK


def test_forward_to_operand():
    def call(p=Y, s=S, m=M, r=R):
        return hk.lib.mxfp6_layer_norm_quantize(X, 0, W, B, 0, hk.E4M3, p, s, m, r, ROWS, H, 1e-5, None)

    for at in (W, B, M, R, S):
        assert _refused(call(p=at)) and _refused(call(p=at - ROWS * H + 16))
    for at in (W, B, M, R):
        assert _refused(call(s=at)) and _refused(call(s=at - 1))
    for at in (X, W, B, Y, S):
        assert _refused(call(m=at)) and _refused(call(r=at))


def test_gradient():
    def call(dx=Y, w=W, m=M, r=R):
        return hk.lib.mxfp6_layer_norm_backward(B, X, 0, m, r, w, 0, dx, None, None, ROWS, H, None, 0, None)

    span = ROWS * H * 4
    for at, size in ((W, 4 * H), (M, 4 * ROWS), (R, 4 * ROWS)):
        for dx in (at, at - span + 4, at + size - 4):
            assert _refused(call(dx=dx)), (at, dx)
