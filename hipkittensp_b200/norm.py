"""Layer norm in front of a projection: the result in x's type or as an MX operand for the GEMM, and the gradient.

The tensors are torch's (device memory and streams only); the kernels are behind the C ABI (mxfp6_layer_norm*).
"""
from __future__ import annotations

import torch

from ._lib import E2M3, lib
from .gemm import _launch, row_bytes

_DTYPE = {torch.float32: 0, torch.bfloat16: 1}


def _rows_matrix(t, name: str) -> None:
    if not isinstance(t, torch.Tensor):
        raise RuntimeError("Expected a torch.Tensor")
    if not t.is_contiguous():
        raise RuntimeError("Tensor must be contiguous")
    if not t.is_cuda:
        raise RuntimeError("Tensor must be on CUDA device")
    if t.dtype not in _DTYPE or t.dim() != 2:
        raise RuntimeError(f"{name} must be a 2-D fp32 or bf16 tensor")
    if t.shape[1] < 1:
        raise RuntimeError(f"{name} must have at least one column")


def _vector(t, name: str, n: int, like, dtype=None) -> int:
    """Checks an optional vector of n elements on like's device; its address (0 if absent)."""
    if t is None:
        return 0
    if not isinstance(t, torch.Tensor):
        raise RuntimeError("Expected a torch.Tensor")
    if not t.is_contiguous():
        raise RuntimeError("Tensor must be contiguous")
    if not t.is_cuda or t.get_device() != like.get_device():
        raise RuntimeError("all tensors must be on the same device")
    if t.dtype not in (_DTYPE if dtype is None else (dtype,)):
        raise RuntimeError(f"{name} must be {'fp32 or bf16' if dtype is None else dtype}")
    if t.dim() != 1 or t.shape[0] != n:
        raise RuntimeError(f"{name} must have {n} elements")
    return t.data_ptr()


def _parameters(x, weight, bias):
    H = x.shape[1]
    w, b = _vector(weight, "weight", H, x), _vector(bias, "bias", H, x)
    if weight is not None and bias is not None and weight.dtype != bias.dtype:
        raise RuntimeError("weight and bias must have the same dtype")
    p = weight if weight is not None else bias
    return w, b, 0 if p is None else _DTYPE[p.dtype]


def layer_norm(x, weight=None, bias=None, eps: float = 1e-5, out=None):
    """y = (x - mean) * rstd * weight + bias over each row of x [rows, H] (fp32 or bf16), in fp32, rounded once to x's type.

    weight and bias [H] (fp32 or bf16, the same type) may be None.  Returns (y, mean, rstd), the statistics fp32 [rows] as
    layer_norm_backward takes them; `out` (may be x) receives y."""
    _rows_matrix(x, "x")
    rows, H = x.shape
    w, b, wd = _parameters(x, weight, bias)
    if out is None:
        out = torch.empty_like(x)
    else:
        _rows_matrix(out, "out")
        if out.shape != x.shape or out.dtype != x.dtype or out.get_device() != x.get_device():
            raise RuntimeError("out must have the shape, dtype and device of x")
    mean = x.new_empty(rows, dtype=torch.float32)
    rstd = torch.empty_like(mean)
    _launch(x, lib.mxfp6_layer_norm, x.data_ptr(), _DTYPE[x.dtype], w, b, wd, out.data_ptr(), mean.data_ptr(), rstd.data_ptr(),
            rows, H, eps)
    return out, mean, rstd


def layer_norm_quantize(x, weight=None, bias=None, eps: float = 1e-5, fmt: int = E2M3):
    """layer_norm whose result leaves as an MX operand for the product that follows (blocks of 32 along H, H % 32 == 0), rounded
    once from fp32 by the rule of quantize().  Returns (operand bytes, scales [rows, H/32], mean, rstd)."""
    _rows_matrix(x, "x")
    rows, H = x.shape
    if H % 32:
        raise RuntimeError("H must be a multiple of 32")
    w, b, wd = _parameters(x, weight, bias)
    packed = x.new_empty((rows, row_bytes(H, fmt)), dtype=torch.uint8)
    scales = x.new_empty((rows, H // 32), dtype=torch.uint8)
    mean = x.new_empty(rows, dtype=torch.float32)
    rstd = torch.empty_like(mean)
    _launch(x, lib.mxfp6_layer_norm_quantize, x.data_ptr(), _DTYPE[x.dtype], w, b, wd, fmt, packed.data_ptr(), scales.data_ptr(),
            mean.data_ptr(), rstd.data_ptr(), rows, H, eps)
    return packed, scales, mean, rstd


def _backward(dy, x, m, r, w, wd, dx, dweight, dbias, stream) -> int:
    rows, H = x.shape
    nbytes = lib.mxfp6_layer_norm_backward_workspace_bytes(rows, H)
    work = x.new_empty(nbytes, dtype=torch.uint8)
    return lib.mxfp6_layer_norm_backward(dy.data_ptr(), x.data_ptr(), _DTYPE[x.dtype], m, r, w, wd, dx.data_ptr(), dweight.data_ptr(),
                                         dbias.data_ptr(), rows, H, work.data_ptr(), nbytes, stream)


def layer_norm_backward(dy, x, mean, rstd, weight=None):
    """Gradient of layer_norm: dy and x [rows, H] of one type, mean and rstd from the forward pass.

    Returns (dx, dweight, dbias): dx in x's type, the sums over the rows in fp32 [H] whatever weight's type."""
    _rows_matrix(x, "x")
    _rows_matrix(dy, "dy")
    if dy.shape != x.shape or dy.dtype != x.dtype or dy.get_device() != x.get_device():
        raise RuntimeError("dy must have the shape, dtype and device of x")
    rows, H = x.shape
    if mean is None or rstd is None:
        raise RuntimeError("Expected a torch.Tensor")
    m, r = _vector(mean, "mean", rows, x, torch.float32), _vector(rstd, "rstd", rows, x, torch.float32)
    w, _, wd = _parameters(x, weight, None)
    dx = torch.empty_like(x)
    dweight = x.new_empty(H, dtype=torch.float32)
    dbias = torch.empty_like(dweight)
    _launch(x, _backward, dy, x, m, r, w, wd, dx, dweight, dbias)
    return dx, dweight, dbias
