"""The layer norm at widths whose parameters take about 48 KB of shared memory as fp32, the amount from which a kernel needs leave to use it
(counted with its static share), and at the edges between the kernels' variants."""
import pytest
import torch

import hipkittensp_b200 as hk
from tests.test_norm_gpu import _check_backward, _check_forward, _codes_match, _inputs

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("H", [6064, 6096, 6112, 6120, 6121, 6127, 6128, 6129, 6135, 6136, 6143, 6144, 6145, 6151, 6152, 6160])
def test_rows_of_about_6144(H, dtype):
    x, w, b, dy = _inputs(40, H, dtype)
    y, mean, rstd = hk.layer_norm(x, w, b)
    assert torch.isfinite(y).all()
    _check_forward(x, w, b, 1e-5, y, mean, rstd)
    _check_backward(dy, x, mean, rstd, w, *hk.layer_norm_backward(dy, x, mean, rstd, w))


@pytest.mark.parametrize("fmt", [hk.E2M3, hk.E3M2, hk.E4M3, hk.E5M2, hk.E2M1])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("H", [6112, 6144, 6176])
def test_rows_of_about_6144_to_operand(H, dtype, fmt):
    x, w, b, _ = _inputs(21, H, dtype, torch.float32)
    packed, scales, mean, rstd = hk.layer_norm_quantize(x, w, b, fmt=fmt)
    _check_forward(x, w, b, 1e-5, None, mean, rstd)
    _codes_match(x, w, b, fmt, packed, scales)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_every_width_is_accepted(dtype):
    """One call each of all widths up to 1100, and of those beside every multiple of 256 up to the longest rows that registers hold."""
    widths = list(range(1, 1101)) + [w + d for w in range(1280, 16641, 256) for d in (-8, -7, -1, 0, 1, 8)]
    buf = torch.randn(3 * max(widths), device="cuda", generator=torch.Generator(device="cuda").manual_seed(1)).to(dtype)
    for H in widths:
        x = buf[:3 * H].view(3, H)
        y, mean, rstd = hk.layer_norm(x)
        want = torch.nn.functional.layer_norm(x.double(), (H,))
        assert (y.double() - want).abs().max() <= 0.03, H            # (bf16 half steps of values up to 4; what is looked for is a refusal)
        hk.layer_norm_backward(x, x, mean, rstd)
        if H % 32 == 0:
            hk.layer_norm_quantize(x, fmt=hk.E4M3)
    assert hk.device_status() == 0
