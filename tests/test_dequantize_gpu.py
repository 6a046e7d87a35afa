"""The streaming dequantiser where its rings go round: at least eight tiles of 64 blocks for every warp that is resident, with a ragged tail,
bit for bit against the plain kernel; and block counts around one tile against the oracle."""
import numpy as np
import pytest
import torch

import hipkittensp_b200 as hk
from oracle import mxfp6_ref as R

pytestmark = pytest.mark.gpu

FORMATS = [R.E2M3, R.E3M2, R.E4M3, R.E5M2, R.E2M1]


@pytest.fixture(autouse=True)
def _clean_options():
    yield
    hk.debug_option("MXFP6_QUANT_PATH", None)


def _ints(t):
    return t.view(torch.int32 if t.dtype == torch.float32 else torch.int16)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("fmt", FORMATS)
def test_many_tiles_per_warp(fmt, dtype):
    sms = torch.cuda.get_device_properties(0).multi_processor_count
    K = 32 * 223
    rows = -(-8 * sms * 6 * 4 * 64 // 223) + 3                  # six CTAs of four warps an SM at most
    assert rows * 223 % 64 and rows * 223 >= 8 * sms * 6 * 4 * 64
    g = torch.Generator(device="cuda").manual_seed(fmt)
    packed = torch.randint(0, 256, (rows, R._FMT[fmt]["bits"] * K // 8), dtype=torch.uint8, device="cuda", generator=g)
    scales = torch.randint(0, 256, (rows, K // 32), dtype=torch.uint8, device="cuda", generator=g)
    got = hk.dequantize(packed, scales, fmt, dtype=dtype)
    hk.debug_option("MXFP6_QUANT_PATH", "quad")
    want = hk.dequantize(packed, scales, fmt, dtype=dtype)
    assert hk.device_status() == 0
    assert torch.equal(_ints(got), _ints(want))
    # ... and the plain kernel against the oracle, on rows of the beginning, the middle and the end
    for at in (0, rows // 2, rows - 2):
        ref = torch.from_numpy(R.dequantize(packed[at:at + 2].cpu().numpy(), scales[at:at + 2].cpu().numpy(), fmt)).to(dtype)
        have = got[at:at + 2].cpu()
        nan = torch.isnan(ref)
        assert torch.equal(torch.isnan(have), nan) and torch.equal(_ints(have)[~nan], _ints(ref)[~nan])


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("blocks", [1, 31, 63, 64, 65, 127, 128, 129, 255, 256, 257])
def test_block_counts_around_a_tile(blocks, fmt, dtype):
    rng = np.random.default_rng(blocks)
    packed = rng.integers(0, 256, size=(1, R._FMT[fmt]["bits"] * blocks * 4), dtype=np.uint8)
    scales = rng.integers(0, 255, size=(1, blocks), dtype=np.uint8)
    want = torch.from_numpy(R.dequantize(packed, scales, fmt)).to(dtype)
    got = hk.dequantize(torch.from_numpy(packed).cuda(), torch.from_numpy(scales).cuda(), fmt, dtype=dtype).cpu()
    assert hk.device_status() == 0
    nan = torch.isnan(want)
    assert torch.equal(torch.isnan(got), nan) and torch.equal(_ints(got)[~nan], _ints(want)[~nan])
