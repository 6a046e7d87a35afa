"""MX-FP4 (E2M1) on the CPU: the oracle against the CUDA toolkit's conversions and the format's rules, and what the entry
points refuse before they touch a device."""
import json
import os

import numpy as np
import pytest
import torch

import hipkittensp_b200 as hk
from hipkittensp_b200 import _lib
from oracle import mxfp6_ref as R

KAT = os.path.join(os.path.dirname(__file__), "golden", "toolkit_fp4_kat.json")


@pytest.fixture(scope="module")
def kat():
    with open(KAT) as f:
        return json.load(f)


def test_oracle_elements_match_the_toolkit(kat):
    enc = np.array(kat["encode"], dtype=np.uint32)
    x = enc[:, 0].copy().view(np.float32)
    np.testing.assert_array_equal(R.encode_elems(x, R.E2M1), enc[:, 1].astype(np.uint8))
    L = R.c_oracle()
    np.testing.assert_array_equal(np.array([L.mxfp6_encode_elem(float(v), R.E2M1) for v in x], np.uint8), enc[:, 1].astype(np.uint8))
    np.testing.assert_array_equal(R.decode_table(R.E2M1).view(np.uint32), np.array(kat["decode"], np.uint32))
    assert R.decode_table(R.E2M1)[:8].tolist() == [0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0]
    lo, hi, byte = kat["pair"]
    pair = R.encode_elems(np.array([lo, hi], np.uint32).view(np.float32), R.E2M1)
    assert R.pack_nibbles(pair).tolist() == [byte]


@pytest.mark.parametrize("config", ["normal", "lognormal", "ffn", "decode"])
def test_oracle_blocks_numpy_equals_c(config):
    for x in R.make_inputs(config, 24, 40, 256, seed=3):
        p1, s1 = R.quantize(x, R.E2M1)
        p2, s2 = R.c_quantize(x, R.E2M1)
        assert p1.shape == (x.shape[0], 128)
        np.testing.assert_array_equal(s1, s2)
        np.testing.assert_array_equal(p1, p2)
        np.testing.assert_array_equal(R.dequantize(p1, s1, R.E2M1), R.c_dequantize(p1, s1, R.E2M1))
        # largest element of a block of scale 2^e lies in [4, 8) * 2^e: the code is 4 or 6
        d = np.abs(R.dequantize(p1, s1, R.E2M1)).reshape(-1, 32).max(1) / R.e8m0_decode(s1).reshape(-1)
        assert set(np.unique(d)) <= {4.0, 6.0}


def test_python_wrappers_refuse():
    A, C, S = torch.zeros(16, 64, dtype=torch.uint8), torch.zeros(16, 16, dtype=torch.bfloat16), torch.zeros(16, 4, dtype=torch.uint8)
    with pytest.raises(RuntimeError, match="Tensor must be on CUDA device"):
        hk.dispatch_micro(A, A, C, S, S, hk.E2M1)
    with pytest.raises(RuntimeError, match="Tensor must be on CUDA device"):
        hk.dequantize(A, S, hk.E2M1)
    with pytest.raises(RuntimeError, match="Tensor must be on CUDA device"):
        hk.quantize(torch.zeros(4, 64), hk.E2M1)


def test_c_entry_points_refuse_without_a_device():
    L = hk.lib
    assert L.mxfp6_gemm(None, None, None, None, None, 16, 16, 100, 4, 4, None) == _lib.ERR_BAD_ARG
    assert L.mxfp6_gemm(None, None, None, None, None, 16, 16, 128, 5, 4, None) == _lib.ERR_BAD_ARG
    assert b"MXFP4_E2M1 (4)" in L.mxfp6_last_error()
    assert L.mxfp6_gemm(None, None, None, None, None, 0, 16, 128, 4, 2, None) == _lib.OK
    # operands of 4-bit codes start on 32 bytes like those of 6-bit codes
    assert L.mxfp6_gemm(16, 32, 32, 32, 32, 16, 16, 128, 4, 4, None) == _lib.ERR_BAD_ARG
    assert b"32-byte aligned" in L.mxfp6_last_error()
    assert L.mxfp6_quantize(None, 0, 4, 33, 4, None, None, None) == _lib.ERR_BAD_ARG
    assert L.mxfp6_quantize(None, 0, 4, 32, 5, None, None, None) == _lib.ERR_BAD_ARG
    assert L.mxfp6_quantize(None, 0, 0, 32, 4, None, None, None) == _lib.OK
    assert L.mxfp6_dequantize_ex(None, None, 4, 32, 4, None, 2, None) == _lib.ERR_BAD_ARG
    assert b"out_dtype" in L.mxfp6_last_error()
    assert L.mxfp6_dequantize_ex(32, 32, 4, 32, 4, 8, 1, None) == _lib.ERR_BAD_ARG
    assert b"16-byte aligned" in L.mxfp6_last_error()
    assert L.mxfp6_dequantize_ex(None, None, 0, 32, 4, None, 1, None) == _lib.OK
    assert L.mxfp6_gemm_requant(None, None, None, None, 256, 256, 64, 96, 128, 0, 0, 4, None) == _lib.ERR_BAD_ARG
    assert b"multiple of 64" in L.mxfp6_last_error()
