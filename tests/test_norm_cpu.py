"""What the layer-norm entry points refuse before they touch a device."""
import pytest
import torch

import hipkittensp_b200 as hk
from hipkittensp_b200 import _lib


def test_c_entry_points_refuse_without_a_device():
    L, BAD = hk.lib, _lib.ERR_BAD_ARG
    P = 1 << 20        # an aligned address that no call below may reach

    def fwd(x=P, xd=0, w=P, b=P, wd=0, y=P, rows=4, H=64, eps=1e-5):
        return L.mxfp6_layer_norm(x, xd, w, b, wd, y, P, P, rows, H, eps, None)

    assert fwd(rows=0) == _lib.OK
    for kw, msg in ((dict(rows=-1), b"rows"), (dict(H=0), b"H="), (dict(xd=2), b"dtype"), (dict(wd=3), b"w_dtype"), (dict(eps=-1.0), b"eps"),
                    (dict(eps=float("nan")), b"eps"), (dict(eps=float("inf")), b"eps"), (dict(x=None), b"null"), (dict(y=None), b"null"),
                    (dict(x=P + 2), b"misaligned"), (dict(xd=1, x=P + 1), b"misaligned"), (dict(w=P + 2), b"misaligned"),
                    (dict(rows=1 << 40), b"too large")):
        assert fwd(**kw) == BAD, kw
        assert msg in L.mxfp6_last_error(), (kw, L.mxfp6_last_error())

    def quant(x=P, xd=0, w=P, wd=0, fmt=4, packed=P, scales=P, rows=4, H=64):
        return L.mxfp6_layer_norm_quantize(x, xd, w, w, wd, fmt, packed, scales, P, P, rows, H, 1e-5, None)

    assert quant(rows=0) == _lib.OK
    for kw, msg in ((dict(fmt=5), b"format"), (dict(fmt=-1), b"format"), (dict(H=48), b"multiple of 32"), (dict(packed=None), b"null"), (dict(scales=None), b"null"),
                    (dict(x=P + 16), b"aligned"), (dict(xd=1, x=P + 8), b"aligned"), (dict(w=P + 4), b"aligned"), (dict(packed=P + 8), b"aligned")):
        assert quant(**kw) == BAD, kw
        assert msg in L.mxfp6_last_error(), (kw, L.mxfp6_last_error())

    def bwd(dy=P, x=P, xd=0, mean=P, rstd=P, w=P, dx=P, dw=P, db=P, rows=4, H=64):
        return L.mxfp6_layer_norm_backward(dy, x, xd, mean, rstd, w, 0, dx, dw, db, rows, H, P, 1 << 30, None)

    for kw, msg in ((dict(rows=-1), b"rows"), (dict(H=0), b"H="), (dict(xd=5), b"dtype"), (dict(dy=None), b"null"), (dict(mean=None), b"null"),
                    (dict(dx=None), b"null"), (dict(dy=P + 2), b"misaligned"), (dict(dw=P + 2), b"misaligned"), (dict(rstd=P + 1), b"misaligned")):
        assert bwd(**kw) == BAD, kw
        assert msg in L.mxfp6_last_error(), (kw, L.mxfp6_last_error())
    assert L.mxfp6_layer_norm_backward_workspace_bytes(0, 64) == 0
    assert L.mxfp6_layer_norm_backward_workspace_bytes(4, 0) == 0


def test_results_over_other_rows_are_refused():
    """A result that lies over its operand, but not row upon row, would be read after it was written."""
    L, BAD = hk.lib, _lib.ERR_BAD_ARG
    P, F = 1 << 20, 1 << 30
    for xd, size in ((0, 4), (1, 2)):
        span = 5 * 64 * size
        for shift in (64 * size, span - size, size, -size, -64 * size, size - span):
            assert L.mxfp6_layer_norm(P, xd, F, F, 0, P + shift, F, F, 5, 64, 1e-5, None) == BAD
            assert b"overlaps" in L.mxfp6_last_error(), shift
            for dy, x in ((P, F), (F, P)):
                assert L.mxfp6_layer_norm_backward(dy, x, xd, F, F, F, 0, P + shift, F, F, 5, 64, F, 1 << 30, None) == BAD
                assert b"overlaps" in L.mxfp6_last_error(), shift
        for packed, scales in ((P, F), (P + span - 16, F), (P - 16, F), (F, P), (F, P + span - 1), (F, P - 9)):
            assert L.mxfp6_layer_norm_quantize(P, xd, F, F, 0, 4, packed, scales, F, F, 5, 64, 1e-5, None) == BAD
            assert b"overlaps" in L.mxfp6_last_error(), (packed, scales)


def test_python_wrappers_refuse():
    x = torch.zeros(4, 64)
    for f in (lambda: hk.layer_norm(x), lambda: hk.layer_norm_quantize(x), lambda: hk.layer_norm_backward(x, x, x[:, 0], x[:, 0])):
        with pytest.raises(RuntimeError, match="Tensor must be on CUDA device"):
            f()
    with pytest.raises(RuntimeError, match="Expected a torch.Tensor"):
        hk.layer_norm([1.0])
    with pytest.raises(RuntimeError, match="Tensor must be contiguous"):
        hk.layer_norm(x.t())
