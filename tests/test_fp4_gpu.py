"""MX-FP4 (E2M1) on the GPU: quantiser and dequantiser bit for bit against the oracle, products against the 64-bit product of the
exactly dequantised operands."""
import numpy as np
import pytest
import torch

import hipkittensp_b200 as hk
from oracle import mxfp6_ref as R
from tests.gpu_util import check, oracle_f64, quantized_inputs, run_gpu

pytestmark = pytest.mark.gpu

FP4 = R.E2M1


@pytest.fixture(autouse=True)
def _clean_options():
    yield
    for name in ("MXFP6_FORCE_CFG", "MXFP6_NO_SF_TMA", "MXFP6_QUANT_PATH", "MXFP6_F4"):
        hk.debug_option(name, None)


def _bits(t):
    return t.contiguous().view(torch.int32 if t.dtype == torch.float32 else torch.int16).cpu().numpy()


# ---------------------------------------------------------------------------------- quantiser, dequantiser
@pytest.mark.parametrize("path", ["stream", "quad"])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("rows,K", [(1, 32), (5, 96), (3, 32 * 43), (129, 32), (1000, 2464), (2048, 4096)])
def test_quantize_bit_exact(path, dtype, rows, K):
    if path == "quad":
        hk.debug_option("MXFP6_QUANT_PATH", "quad")
    g = torch.Generator().manual_seed(rows + K)
    x = (torch.randn(rows, K, generator=g).reshape(-1, 32) * torch.exp(torch.randn(rows * K // 32, 1, generator=g))).reshape(rows, K).to(dtype)
    pa, sa = R.c_quantize(np.ascontiguousarray(x.float().numpy()), FP4)
    gp, gs = hk.quantize(x.cuda(), hk.E2M1)
    assert hk.device_status() == 0
    np.testing.assert_array_equal(gs.cpu().numpy(), sa)
    np.testing.assert_array_equal(gp.cpu().numpy(), pa)


@pytest.mark.parametrize("path", ["stream", "quad"])
def test_quantize_edge_values(path):
    """Zero and signed-zero blocks, the saturation gap (6, 8), ties, subnormal and huge blocks, infinities."""
    if path == "quad":
        hk.debug_option("MXFP6_QUANT_PATH", "quad")
    x = np.zeros((8, 256), np.float32)
    x[1, :32] = 1.0
    x[2, :8] = [7.9, 6.0, 5.0, 3.5, 2.5, 1.75, 1.25, 0.25]
    x[3, :32] = 1e-30
    x[4, 5] = -0.0
    x[5, :64] = np.linspace(-100, 100, 64)
    x[6, :] = np.ldexp(1.0, -140)
    x[7, ::2] = 3.0e38
    x[7, 200] = np.inf
    pa, sa = R.quantize(x, FP4)
    gp, gs = hk.quantize(torch.from_numpy(x).cuda(), hk.E2M1)
    np.testing.assert_array_equal(gs.cpu().numpy(), sa)
    np.testing.assert_array_equal(gp.cpu().numpy(), pa)


@pytest.mark.parametrize("fmt", [R.E2M3, R.E3M2, R.E4M3, R.E5M2, R.E2M1])
@pytest.mark.parametrize("rows,K,shift", [(40, 544, 0), (40, 544, 1), (1, 32, 0), (3, 32, 0), (1, 1056, 0), (700, 2048, 0), (700, 2048, 16)])
def test_dequantize_all_codes_and_scales(fmt, rows, K, shift):
    """Every code under scales over the whole range, to fp32 and bf16; block counts around a warp's tile of 32 and past a ring's
    length; operands that start on an odd byte too."""
    rng = np.random.default_rng(fmt)
    packed = rng.integers(0, 256, size=(rows, R._FMT[fmt]["bits"] * K // 8), dtype=np.uint8)
    scales = rng.integers(1, 255, size=(rows, K // 32), dtype=np.uint8)
    scales.reshape(-1)[:min(3, scales.size)] = [0, 254, 127][:min(3, scales.size)]
    want = torch.from_numpy(R.dequantize(packed, scales, fmt))
    buf = torch.zeros(packed.size + 16, dtype=torch.uint8, device="cuda")
    dev = buf[shift:shift + packed.size].view(rows, -1)
    dev.copy_(torch.from_numpy(packed))
    for dtype in (torch.float32, torch.bfloat16):
        got = hk.dequantize(dev, torch.from_numpy(scales).cuda(), fmt, dtype=dtype)
        assert got.dtype == dtype
        nan = torch.isnan(want)
        assert torch.equal(torch.isnan(got.cpu()), nan)
        w = want.to(dtype)
        np.testing.assert_array_equal(_bits(got)[~nan.numpy()], _bits(w)[~nan.numpy()])


def test_round_trip_large():
    x = torch.randn(8192, 8192, device="cuda", generator=torch.Generator(device="cuda").manual_seed(3))
    p, s = hk.quantize(x, hk.E2M1)
    for dtype in (torch.float32, torch.bfloat16):
        p2, s2 = hk.quantize(hk.dequantize(p, s, hk.E2M1, dtype=dtype), hk.E2M1)
        assert torch.equal(p, p2) and torch.equal(s, s2)


# ---------------------------------------------------------------------------------- products
PAIRS = [(FP4, FP4), (R.E4M3, FP4), (R.E2M3, FP4), (FP4, R.E5M2), (FP4, R.E3M2)]
# (M, N, K): one token, the swapped forms and their tile edges, wide unswapped tiles, single-CTA tiles, the CTA pair with ragged
# rows, columns and K; K / 128 odd and even, scale rows that are and are not 16-byte multiples
SHAPES = [(1, 28672, 256), (16, 24320, 384), (16, 520, 1024), (17, 384, 640), (33, 200, 128), (64, 24000, 256), (100, 30000, 128), (128, 130, 2048),
          (130, 200, 384), (300, 520, 1152), (384, 768, 512), (1536, 1792, 640), (1111, 2050, 1024), (2048, 2304, 256),
          # rows of C that are not 16-byte multiples, odd and even, in the unswapped single-CTA tiles
          # even-rows tiles of few rows per CTA, ragged in rows and columns
          (3, 14400, 512), (16, 19500, 4224), (32, 15001, 1024),
          (300, 1001, 512), (300, 1002, 384), (70, 30001, 128), (520, 1003, 256)]


def _run(M, N, K, fa, fb, force=None, seed=0, config="lognormal"):
    if force:
        hk.debug_option("MXFP6_FORCE_CFG", force)
    pa, sa, pb, sb = quantized_inputs(config, M, N, K, fa, seed, fb)
    c = run_gpu(pa, sa, pb, sb, fa, fb)
    ref, absdot = oracle_f64(pa, sa, pb, sb, fa, fb)
    return check(c, ref, absdot)


@pytest.mark.parametrize("pair", PAIRS)
@pytest.mark.parametrize("shape", SHAPES)
def test_products(shape, pair):
    _run(*shape, *pair, seed=sum(shape))


@pytest.mark.parametrize("shape", SHAPES)
def test_products_on_spread_nibbles(shape):
    """Two E2M1 operands on the 8-bit path of the mixed pairs: the same sums."""
    hk.debug_option("MXFP6_F4", "0")
    _run(*shape, FP4, FP4, seed=sum(shape))


@pytest.mark.parametrize("shape", [(16, 512, 1024), (64, 640, 384), (130, 200, 1152)])
def test_caller_workspace(shape):
    """mxfp6_gemm_ws with exactly the bytes the library asks for, on the 4-bit path and with a mixed pair."""
    M, N, K = shape
    need = hk.lib.mxfp6_gemm_workspace_bytes(M, N, K)
    for fa in (FP4, R.E4M3):
        pa, sa, pb, sb = quantized_inputs("normal", M, N, K, fa, 1, FP4)
        t = [torch.from_numpy(x).cuda() for x in (pa, sa, pb, sb)]
        ws, C = torch.zeros(max(need, 1), dtype=torch.uint8, device="cuda"), torch.empty(M, N, dtype=torch.bfloat16, device="cuda")
        rc = hk.lib.mxfp6_gemm_ws(*[x.data_ptr() for x in t], C.data_ptr(), M, N, K, fa, FP4, ws.data_ptr(), need, torch.cuda.current_stream().cuda_stream)
        assert rc == 0, hk.lib.mxfp6_last_error()
        assert hk.device_status() == 0
        check(C.float().cpu().numpy(), *oracle_f64(pa, sa, pb, sb, fa, FP4))


@pytest.mark.parametrize("fa", [FP4, R.E4M3])
def test_side_by_side_with_a_workspace_each(fa):
    """Products whose tiles are split along K: on two streams at once, then in two captured graphs replayed at once."""
    M, N, K = 16, 512, 8192
    assert hk.gemm_workspace(M, N, K).numel() > 0
    sides = []
    for seed in (1, 2):
        host = quantized_inputs("normal", M, N, K, fa, seed, FP4)
        out = torch.empty(24, M, N, dtype=torch.bfloat16, device="cuda")
        sides.append((host, [torch.from_numpy(x).cuda() for x in host], hk.gemm_workspace(M, N, K), out, torch.cuda.Stream()))
    torch.cuda.synchronize()

    def verify():
        torch.cuda.synchronize()
        assert hk.device_status() == 0
        for host, _, _, out, _ in sides:
            assert (out == out[0]).all()
            check(out[0].float().cpu().numpy(), *oracle_f64(*host, fa, FP4))
            out.zero_()
        torch.cuda.synchronize()

    for i in range(24):
        for _, t, ws, out, stream in sides:
            with torch.cuda.stream(stream):
                hk.gemm(*t, fmt=fa, fmt_b=FP4, out=out[i], workspace=ws)
    verify()
    graphs = []
    for _, t, ws, out, _ in sides:
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[-1]):
            for i in range(24):
                hk.gemm(*t, fmt=fa, fmt_b=FP4, out=out[i], workspace=ws)
    for graph, (*_, stream) in zip(graphs, sides):
        with torch.cuda.stream(stream):
            graph.replay()
    verify()


def test_workspace_refusals():
    t = [torch.from_numpy(x).cuda() for x in quantized_inputs("normal", 16, 512, 8192, FP4, 1)]
    ws = hk.gemm_workspace(16, 512, 8192)
    for bad in (ws[:1024], ws[8:], ws.cpu(), ws.view(torch.float32), ws[::2], 7):
        with pytest.raises(RuntimeError):
            hk.gemm(*t, fmt=FP4, workspace=bad)
    assert hk.gemm_workspace(4096, 4096, 1024).numel() == 0


@pytest.mark.parametrize("pair", PAIRS[:2])
@pytest.mark.parametrize("force", ["128,0,0", "256,0,0", "128,0,1", "256,0,1", "16,1,0", "32,1,1", "64,1,1", "128,1,1", "256,0,0,1"])
def test_kernel_variants(force, pair):
    M = 16 if force.startswith("16,1") else 30 if force.startswith("32,1") else 60 if force.startswith("64,1") else 100 if force.startswith("128,1") else 384
    _run(M, 768, 896, *pair, force=force, seed=1)


@pytest.mark.parametrize("pair", PAIRS[:2])
@pytest.mark.parametrize("force", ["128,0,0", "256,0,0,1", "32,1,1"])
def test_plain_scale_loads(force, pair):
    hk.debug_option("MXFP6_NO_SF_TMA", "1")
    _run(30 if force.startswith("32,1") else 300, 512, 1024, *pair, force=force, seed=4)


@pytest.mark.parametrize("shape", [(16, 512, 512), (256, 512, 512), (2048, 2048, 512)])
def test_one_hot_operand_exposes_layout(shape):
    """One-hot rows of B pick elements of A exactly: any mistake in the operand or scale layout moves or rescales them."""
    M, N, K = shape
    A, _ = R.make_inputs("lognormal", M, N, K, seed=5)
    pa, sa = R.quantize(A, FP4)
    pb, sb = R.quantize(np.eye(N, K, k=0, dtype=np.float32) if N <= K else np.tile(np.eye(K, dtype=np.float32), (N // K, 1)), FP4)
    c = run_gpu(pa, sa, pb, sb, FP4)
    want = R.dequantize(pa, sa, FP4)[:, np.arange(N) % K]
    np.testing.assert_array_equal(c, want)


@pytest.mark.parametrize("shape", [(16, 640, 1024), (300, 520, 640), (2048, 2304, 384)])
def test_scaled_epilogue(shape):
    M, N, K = shape
    pa, sa, pb, sb = quantized_inputs("normal", M, N, K, FP4, 2)
    rng = np.random.default_rng(0)
    row, col, bias = (rng.normal(1, 0.2, n).astype(np.float32) for n in (M, N, N))
    t = [torch.from_numpy(x).cuda() for x in (pa, sa, pb, sb, row, col, bias)]
    c = hk.gemm_scaled(*t, fmt=hk.E2M1).float().cpu().numpy()
    assert hk.device_status() == 0
    ref, absdot = oracle_f64(pa, sa, pb, sb, FP4)
    s = row[:, None].astype(np.float64) * col[None, :]
    check(c, ref * s + bias, absdot * np.abs(s) + np.abs(bias))


@pytest.mark.parametrize("out_fmt", [R.E2M1, R.E2M3, R.E4M3])
@pytest.mark.parametrize("fa,fb", [(FP4, FP4), (R.E2M3, R.E2M3), (R.E4M3, FP4)])
@pytest.mark.parametrize("shape", [(1, 24320, 256), (16, 640, 1024), (100, 24064, 128), (300, 576, 640), (2048, 2304, 384)])
def test_requantised_result(shape, fa, fb, out_fmt):
    """The requantising epilogue rounds the fp32 sum of the same kernel that writes bf16: against the quantised 64-bit product the
    scale may differ where the block's largest value lies at a power of two, and a code by one step where the value lies at a
    rounding boundary; every decoded value is within one step of its block of the 64-bit product."""
    M, N, K = shape
    pa, sa, pb, sb = quantized_inputs("normal", M, N, K, fa, 3, fb)
    t = [torch.from_numpy(x).cuda() for x in (pa, sa, pb, sb)]
    out, scales = hk.gemm_requant(*t, fmt=fa, fmt_b=fb, out_fmt=out_fmt)
    assert hk.device_status() == 0
    ref, absdot = oracle_f64(pa, sa, pb, sb, fa, fb)
    wp, ws = R.quantize(ref.astype(np.float32), out_fmt)
    gp, gs = out.cpu().numpy(), scales.cpu().numpy()
    same = gs == ws
    assert same.mean() > 0.999 and np.abs(gs.astype(int) - ws).max() <= 1
    got, want = R.codes_of(gp, out_fmt).reshape(M, N // 32, 32)[same], R.codes_of(wp, out_fmt).reshape(M, N // 32, 32)[same]
    differ = got != want
    assert differ.mean() < 1e-3
    d, w = R.dequantize(gp, gs, out_fmt), R.dequantize(wp, ws, out_fmt)
    mant, emax = R._FMT[out_fmt]["mbits"], R._FMT[out_fmt]["emax"]
    step = np.ldexp(1.0, np.maximum(gs, ws).astype(int) - 127 + emax - mant).repeat(32, axis=1)
    assert (np.abs(d - w) <= step).all()


def test_several_destinations():
    M, N, K = 512, 768, 384
    pa, sa, pb, sb = quantized_inputs("normal", M, N, K, FP4, 4)
    t = [torch.from_numpy(x).cuda() for x in (pa, sa, pb, sb)]
    dests = [torch.zeros(M, N + 64, dtype=torch.bfloat16, device="cuda") for _ in range(3)]
    hk.dispatch_multi(t[0], t[2], dests, 32, t[1], t[3], hk.E2M1)
    want = hk.gemm(t[0], t[1], t[2], t[3], hk.E2M1)
    assert hk.device_status() == 0
    for d in dests:
        assert torch.equal(d[:, 32:32 + N], want) and not d[:, :32].any() and not d[:, 32 + N:].any()


def test_host_pipeline_and_extension_module():
    import os
    import sys
    M, N, K = 64, 512, 256
    pa, sa, pb, sb = quantized_inputs("normal", M, N, K, FP4, 6)
    ref, absdot = oracle_f64(pa, sa, pb, sb, FP4)
    pin = [torch.from_numpy(x).pin_memory() for x in (pa, sa, pb, sb)]
    out = torch.empty(M, N, dtype=torch.bfloat16).pin_memory()
    g = hk.HostGemm(M, N, K, fmt=hk.E2M1)
    g(*pin, out)
    g.synchronize()
    check(out.float().numpy(), ref, absdot)
    sys.path.insert(0, os.path.dirname(hk.__file__))
    import tk_kernel
    C = torch.empty(M, N, dtype=torch.bfloat16, device="cuda")
    t = [x.cuda() for x in pin]
    tk_kernel.dispatch_micro(t[0], t[2], C, t[1], t[3], hk.E2M1)
    check(C.float().cpu().numpy(), ref, absdot)
