"""Products written into a column window of a wider matrix: the columns beside the window stay as they were, whatever its width and place."""
import pytest
import torch

import hipkittensp_b200 as hk
from oracle import mxfp6_ref as R

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True)
def _clean_options():
    yield
    for name in ("MXFP6_FORCE_CFG", "MXFP6_C_TMA_LAST"):
        hk.debug_option(name, None)


def _operands(M, N, K, fmt):
    g = torch.Generator(device="cuda").manual_seed(M + N + K)
    n = lambda *s: torch.randn(*s, device="cuda", generator=g)
    return [*hk.quantize(n(M, K), fmt), *hk.quantize(0.05 * n(N, K), fmt)]


def _check(M, N, K, fmt, dests, lead, tail):
    A, sA, B, sB = _operands(M, N, K, fmt)
    want = hk.gemm(A, sA, B, sB, fmt)
    ds = [torch.full((M, lead + N + tail), float("nan"), dtype=torch.bfloat16, device="cuda") for _ in range(dests)]
    hk.dispatch_multi(A, B, ds, lead, sA, sB, fmt)
    assert hk.device_status() == 0
    ref = hk.dequantize(A, sA, fmt).double() @ hk.dequantize(B, sB, fmt).double().t()
    assert ((want.double() - ref).abs() <= 2.0 ** -8 * ref.abs() * 1.02 + 1e-3).all()
    for d in ds:
        assert torch.isnan(d[:, :lead]).all() and torch.isnan(d[:, lead + N:]).all(), "columns beside the window were written"
        # (another kernel may have summed in another order: one bf16 step, and the fp32 noise of sums that cancel)
        assert ((d[:, lead:lead + N].double() - want.double()).abs() <= 2.0 ** -7 * want.double().abs() + 1e-3).all()


@pytest.mark.parametrize("lead,tail", [(0, 3), (8, 11), (64, 3), (3, 5), (0, 4)])
@pytest.mark.parametrize("dests", [1, 3])
# the CTA pair, with and without column slices; single-CTA tiles; wide unswapped tiles; swapped tiles
@pytest.mark.parametrize("M,N,K", [(716, 5005, 256), (1536, 1797, 256), (257, 2563, 128), (300, 573, 384), (200, 261, 256), (100, 30005, 128), (16, 573, 256), (16, 28677, 256), (40, 1021, 512)])
@pytest.mark.parametrize("fmt", [R.E2M3, R.E2M1])
def test_columns_beside_the_window_stay(M, N, K, fmt, dests, lead, tail):
    _check(M, N, K, fmt, dests, lead, tail)


@pytest.mark.parametrize("extra", range(1, 8))
def test_every_ragged_width(extra):
    for M, N in ((300, 1024 + extra), (300, 512 + extra)):
        _check(M, N, 256, R.E2M3, 1, 8, (8 - extra) + 8)


@pytest.mark.parametrize("force", ["128,0,0", "256,0,0", "256,0,0,1", "128,0,1", "32,1,0"])
@pytest.mark.parametrize("last", ["0", "1"])
def test_kernel_variants(force, last):
    hk.debug_option("MXFP6_FORCE_CFG", force)
    hk.debug_option("MXFP6_C_TMA_LAST", last)
    _check(30 if force.startswith("32") else 300, 517, 512, R.E2M3, 1, 8, 3)


def test_a_ragged_window_has_no_completion_flags():
    """The gather by copy engines needs TMA stores of C, which cannot end inside a 16-byte unit: refused."""
    M, N, K = 2048, 1277, 256                            # (enough tiles for the CTA pair)
    A, sA, B, sB = _operands(M, N, K, R.E2M3)
    d = torch.full((M, 1280), float("nan"), dtype=torch.bfloat16, device="cuda")
    scratch = torch.zeros(1024, dtype=torch.int32, device="cuda")
    with pytest.raises(hk.Mxfp6Error, match="multiple of 8"):
        hk.dispatch_copy_gather(A, B, [d], 0, sA, sB, scratch, [])
    torch.cuda.synchronize()
    assert torch.isnan(d).all()
    d8 = torch.full((M, 1288), float("nan"), dtype=torch.bfloat16, device="cuda")
    A, sA, B, sB = _operands(M, 1280, K, R.E2M3)
    hk.dispatch_copy_gather(A, B, [d8], 8, sA, sB, scratch, [])
    assert torch.equal(d8[:, 8:], hk.gemm(A, sA, B, sB)) and torch.isnan(d8[:, :8]).all()


def test_destinations_that_are_no_gpu_memory_are_refused():
    """A matrix in host memory, or no matrix: refused on the host, before anything could write there."""
    M, N, K = 300, 512, 256
    A, sA, B, sB = _operands(M, N, K, R.E2M3)
    good = torch.zeros(M, N, dtype=torch.bfloat16, device="cuda")
    scratch = torch.zeros(1024, dtype=torch.int32, device="cuda")
    for bad in ([good.cpu()], [good, good.cpu()], [good, good.cpu().pin_memory()], [1], [good, None], [good.float()], [good[:100]], [good[:, 1:]], [], [good] * 9):
        with pytest.raises(RuntimeError):
            hk.dispatch_multi(A, B, bad, 0, sA, sB)
        with pytest.raises(RuntimeError):
            hk.dispatch_copy_gather(A, B, bad, 0, sA, sB, scratch, [])
    for bad in (scratch.cpu(), None, scratch[::2]):
        with pytest.raises(RuntimeError):
            hk.dispatch_copy_gather(A, B, [good], 0, sA, sB, bad, [])
    with pytest.raises(RuntimeError, match="Tensor must be on CUDA device"):
        hk.tma_dump(torch.zeros(128, 96, dtype=torch.uint8))
    assert not good.any()
