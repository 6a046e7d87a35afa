"""NaN in re-quantised products: it does not count towards its block's scale, whichever form of the kernel writes the block, and is stored as
the largest magnitude (fp6, fp4) or as NaN (fp8), as the quantiser does."""
import numpy as np
import pytest
import torch

import hipkittensp_b200 as hk
from oracle import mxfp6_ref as R

pytestmark = pytest.mark.gpu

OUT = {hk.E2M3: 0x1f, hk.E3M2: 0x1f, hk.E4M3: 0x7f, hk.E5M2: 0x7f, hk.E2M1: 0x7}      # code of a NaN
# swapped tiles whole and split along K (the wide one by the 128-row form), unswapped tiles, the CTA pair
SHAPES = [(16, 24064, 128), (1, 640, 1024), (16, 640, 1024), (30, 640, 2048), (64, 640, 1024), (120, 640, 1024), (100, 24064, 128), (300, 576, 640), (2048, 2304, 384)]


def _operands(M, N, K, fa, fb):
    g = torch.Generator(device="cuda").manual_seed(M + N + K)
    n = lambda *s: torch.randn(*s, device="cuda", generator=g)
    return [*hk.quantize(n(M, K), fa), *hk.quantize(0.02 * n(N, K), fb)]


@pytest.mark.parametrize("out_fmt", list(OUT))
@pytest.mark.parametrize("fa,fb", [(hk.E4M3, hk.E2M1), (hk.E2M3, hk.E2M3), (hk.E2M1, hk.E2M1)])
@pytest.mark.parametrize("shape", SHAPES)
def test_a_column_of_nan_leaves_its_blocks_alone(shape, fa, fb, out_fmt):
    """One weight row whose scale is NaN, against the same product with that row zero: equal scales, equal codes in the other columns."""
    M, N, K = shape
    A, sA, B, sB = _operands(M, N, K, fa, fb)
    cols = [5, 40, N - 1]
    B[cols] = 0
    want, ws = hk.gemm_requant(A, sA, B, sB, fmt=fa, fmt_b=fb, out_fmt=out_fmt)
    sB[cols, K // 64] = 255
    got, gs = hk.gemm_requant(A, sA, B, sB, fmt=fa, fmt_b=fb, out_fmt=out_fmt)
    assert hk.device_status() == 0
    assert torch.equal(gs, ws)
    g, w = R.codes_of(got.cpu().numpy(), out_fmt), R.codes_of(want.cpu().numpy(), out_fmt)
    assert (g[:, cols] & OUT[out_fmt] == OUT[out_fmt]).all()
    assert np.array_equal(np.delete(g, cols, 1), np.delete(w, cols, 1))


@pytest.mark.parametrize("out_fmt", list(OUT))
@pytest.mark.parametrize("shape", SHAPES)
def test_a_row_of_nan_stays_in_its_row(shape, out_fmt):
    M, N, K = shape
    A, sA, B, sB = _operands(M, N, K, hk.E4M3, hk.E2M1)
    want, ws = hk.gemm_requant(A, sA, B, sB, fmt=hk.E4M3, fmt_b=hk.E2M1, out_fmt=out_fmt)
    row = M // 2
    sA[row, 0] = 255
    got, gs = hk.gemm_requant(A, sA, B, sB, fmt=hk.E4M3, fmt_b=hk.E2M1, out_fmt=out_fmt)
    assert hk.device_status() == 0
    rest = [r for r in range(M) if r != row]
    assert torch.equal(got[rest], want[rest]) and torch.equal(gs[rest], ws[rest])
    assert not gs[row].any()
    assert (R.codes_of(got[row:row + 1].cpu().numpy(), out_fmt) & OUT[out_fmt] == OUT[out_fmt]).all()


@pytest.mark.parametrize("fmt", list(OUT))
@pytest.mark.parametrize("path", ["stream", "quad"])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_the_quantiser_and_nan(fmt, path, dtype):
    hk.debug_option("MXFP6_QUANT_PATH", "quad" if path == "quad" else None)
    try:
        x = torch.randn(64, 256, device="cuda", generator=torch.Generator(device="cuda").manual_seed(1)).to(dtype)
        x[:, 7::32] = 0
        want, ws = hk.quantize(x, fmt)
        x[:, 7::32] = float("nan")
        x[3] = float("nan")
        got, gs = hk.quantize(x, fmt)
    finally:
        hk.debug_option("MXFP6_QUANT_PATH", None)
    rest = [r for r in range(64) if r != 3]
    assert torch.equal(gs[rest], ws[rest]) and not gs[3].any()
    g, w = R.codes_of(got.cpu().numpy(), fmt), R.codes_of(want.cpu().numpy(), fmt)
    nan = np.zeros(256, bool)
    nan[7::32] = True
    assert (g[:, nan] & OUT[fmt] == OUT[fmt]).all() and (g[3] & OUT[fmt] == OUT[fmt]).all()
    assert np.array_equal(g[rest][:, ~nan], w[rest][:, ~nan])
