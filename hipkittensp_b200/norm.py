"""Layer norm in front of a projection: the result in x's type or as an MX operand for the GEMM, and the gradient.

The tensors are torch's (device memory and streams only); the kernels are behind the C ABI (mxfp6_layer_norm*), the argument
checks and the allocation of results in csrc/torch_ops.cpp.
"""
from __future__ import annotations

from ._lib import E2M3, ops


def layer_norm(x, weight=None, bias=None, eps: float = 1e-5, out=None):
    """y = (x - mean) * rstd * weight + bias over each row of x [rows, H] (fp32 or bf16), in fp32, rounded once to x's type.

    weight and bias [H] (fp32 or bf16, the same type) may be None.  Returns (y, mean, rstd), the statistics fp32 [rows] as
    layer_norm_backward takes them; `out` (x itself, or apart from it) receives y."""
    return ops.layer_norm(x, weight, bias, eps, out)


def layer_norm_quantize(x, weight=None, bias=None, eps: float = 1e-5, fmt: int = E2M3):
    """layer_norm whose result leaves as an MX operand for the product that follows (blocks of 32 along H, H % 32 == 0), rounded
    once from fp32 by the rule of quantize().  Returns (operand bytes, scales [rows, H/32], mean, rstd)."""
    return ops.layer_norm_quantize(x, weight, bias, eps, fmt)


def layer_norm_backward(dy, x, mean, rstd, weight=None):
    """Gradient of layer_norm: dy and x [rows, H] of one type, mean and rstd from the forward pass.

    Returns (dx, dweight, dbias): dx in x's type, the sums over the rows in fp32 [H] whatever weight's type."""
    return ops.layer_norm_backward(dy, x, mean, rstd, weight)
