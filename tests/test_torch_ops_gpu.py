"""The compiled wrappers (_torch_ops): what they hold and raise around a call of the library.  The library is replaced by one whose entry
points sleep, or given no memory; no kernel is involved."""
import ctypes
import os
import re
import subprocess
import threading
import time

import pytest
import torch

import hipkittensp_b200 as hk
from hipkittensp_b200 import _lib

pytestmark = pytest.mark.gpu

PKG = os.path.dirname(os.path.abspath(hk.__file__))


@pytest.fixture(scope="module")
def sleeping_library(tmp_path_factory):
    """Every entry point the wrappers use, each taking 0.4 s and doing nothing."""
    src = open(os.path.join(PKG, "csrc", "torch_ops.cpp")).read()
    names = re.findall(r"X\((mxfp6_\w+)\)", src)
    assert "mxfp6_gemm_ws" in names and "mxfp6_layer_norm_backward" in names
    body = "#include <stddef.h>\n#include <unistd.h>\n"
    for n in names:
        if n == "mxfp6_last_error":
            body += f'const char* {n}(void) {{ return "none"; }}\n'
        elif n.endswith("_bytes"):
            body += f"size_t {n}(void) {{ return 256; }}\n"
        else:
            body += f"int {n}(void) {{ usleep(400000); return 0; }}\n"
    d = tmp_path_factory.mktemp("lib")
    c, so = d / "sleep.c", d / "libsleep.so"
    c.write_text(body)
    subprocess.run(["gcc", "-shared", "-fPIC", "-o", str(so), str(c)], check=True)
    return ctypes.CDLL(str(so))


def _calls():
    u8 = lambda *s: torch.zeros(*s, dtype=torch.uint8, device="cuda")
    a, s, x = u8(32, 128), u8(32, 4), torch.zeros(32, 128, device="cuda")
    stat = torch.zeros(32, device="cuda")
    return {
        "gemm": lambda: hk.gemm(a, s, a, s, fmt=hk.E4M3),
        "gemm with a workspace": lambda: hk.gemm(a, s, a, s, fmt=hk.E4M3, workspace=u8(512)),
        "gemm_scaled": lambda: hk.gemm_scaled(a, s, a, s, fmt=hk.E4M3),
        "quantize": lambda: hk.quantize(x),
        "dequantize": lambda: hk.dequantize(a, s, hk.E4M3),
        "layer_norm": lambda: hk.layer_norm(x),
        "layer_norm_quantize": lambda: hk.layer_norm_quantize(x),
        "layer_norm_backward": lambda: hk.layer_norm_backward(x, x, stat, stat),
    }


def test_other_threads_run_while_a_call_waits(sleeping_library):
    """A call that waits in the library lets Python's other threads run: a launch may block on a full queue, whose callbacks may need
    the interpreter."""
    calls = _calls()
    ticks, stop = [], threading.Event()

    def tick():
        while not stop.wait(0.01):
            ticks.append(time.monotonic())

    thread = threading.Thread(target=tick)
    _lib.ops.bind(sleeping_library._handle, _lib.Mxfp6Error)
    try:
        thread.start()
        for name, call in calls.items():
            t0 = time.monotonic()
            call()
            t1 = time.monotonic()
            assert t1 - t0 >= 0.35, name
            # (at most every 10 ms in 400: a quarter of what may be)
            assert sum(t0 + 0.02 < t < t1 - 0.02 for t in ticks) >= 10, f"{name} held the interpreter"
    finally:
        stop.set()
        thread.join()
        _lib.ops.bind(_lib.lib._handle, _lib.Mxfp6Error)
    x = torch.randn(8, 64, device="cuda")
    assert torch.isfinite(hk.layer_norm(x)[0]).all()


def test_out_of_memory_keeps_its_type():
    """A result that does not fit raises torch.OutOfMemoryError, as torch.empty does."""
    codes, scales = torch.zeros(4096, 65536, dtype=torch.uint8, device="cuda"), torch.zeros(4096, 4096, dtype=torch.uint8, device="cuda")
    x = torch.zeros(1 << 16, 4096, device="cuda")
    torch.cuda.empty_cache()
    held = torch.cuda.memory_reserved() + (64 << 20)
    torch.cuda.set_per_process_memory_fraction(held / torch.cuda.get_device_properties(0).total_memory)
    try:
        for call in (lambda: torch.empty(1 << 30, device="cuda"), lambda: hk.dequantize(codes, scales, hk.E2M1), lambda: hk.quantize(x), lambda: hk.layer_norm(x)):
            with pytest.raises(torch.OutOfMemoryError):
                call()
    finally:
        torch.cuda.set_per_process_memory_fraction(1.0)
    assert hk.layer_norm(x[:8])[0].shape == (8, 4096)


def test_gemm_refuses_in_the_words_of_dispatch_micro():
    u8 = lambda *s: torch.zeros(*s, dtype=torch.uint8, device="cuda")
    c = lambda *s: torch.zeros(*s, dtype=torch.bfloat16, device="cuda")
    A, B, sA, sB, C = u8(32, 256), u8(48, 256), u8(32, 8), u8(48, 8), c(32, 48)
    bad = [(1, B, C, sA, sB), (A.t(), B, C, sA, sB), (A.cpu(), B, C, sA, sB), (A.int(), B, C, sA, sB), (A[0], B, C, sA, sB), (A.view(1, 1, 1, 32, 256), B, C, sA, sB),
           (A, 2, C, sA, sB), (A, B.cpu(), C, sA, sB), (A, B, C.float(), sA, sB), (A, B, C, sA.int(), sB), (A, B, C, sA, sB[0]),
           (u8(32, 96), B, C, sA, sB), (A, B, c(31, 48), sA, sB), (A, B, c(32, 47), sA, sB), (A, u8(47, 256), C, sA, sB), (A, u8(48, 128), C, sA, sB),
           (A, B, C, u8(32, 4), sB), (A, B, C, sA, u8(47, 8))]
    for i, (a, b, out, sa, sb) in enumerate(bad):
        texts = []
        for call in (lambda: hk.dispatch_micro(a, b, out, sa, sb, hk.E4M3), lambda: hk.gemm(a, sa, b, sb, hk.E4M3, out=out)):
            with pytest.raises(RuntimeError) as e:
                call()
            texts.append(str(e.value))
        assert texts[0] == texts[1], i
    # fp6 rows that are not whole groups of four codes, and B with another K where the result is allocated
    for call in (lambda: hk.gemm(u8(32, 98), sA, B, sB), lambda: hk.gemm(A, sA, u8(48, 128), sB, hk.E4M3)):
        with pytest.raises(RuntimeError, match="must be 3K/4 bytes|B must be"):
            call()


def test_calls_from_several_threads():
    """Four threads with a stream each, whose calls may now overlap on the host too: the bits of a thread alone."""
    def operands(seed):
        g = torch.Generator(device="cuda").manual_seed(seed)
        n = lambda *s: torch.randn(*s, device="cuda", generator=g)
        x, w, dy = n(24, 1024 + 32 * seed), n(1024 + 32 * seed), n(24, 1024 + 32 * seed)
        B, sB = hk.quantize(0.05 * n(512, 1024), hk.E2M1)
        return x, w, dy, B, sB, hk.gemm_workspace(24, 512, 1024)

    def step(x, w, dy, B, sB, ws):
        A, sA, mean, rstd = hk.layer_norm_quantize(x, w, None, fmt=hk.E2M1)
        y = hk.layer_norm(x, w)[0]
        P, sP = hk.quantize(y[:, :1024].contiguous(), hk.E2M1)
        return (A, sA, y, hk.gemm(P, sP, B, sB, hk.E2M1, workspace=ws), hk.gemm_scaled(P, sP, B, sB, fmt=hk.E2M1, workspace=ws), hk.dequantize(A, sA, hk.E2M1),
                *hk.layer_norm_backward(dy, x, mean, rstd, w))

    cases = [operands(i) for i in range(4)]
    want = [[t.clone() for t in step(*c)] for c in cases]
    torch.cuda.synchronize()
    wrong, errors = [], []

    def work(i):
        try:
            with torch.cuda.stream(torch.cuda.Stream()):
                for k in range(100):
                    got = step(*cases[i])
                    torch.cuda.current_stream().synchronize()
                    if not all(torch.equal(a, b) for a, b in zip(got, want[i])):
                        wrong.append((i, k))
        except BaseException as e:      # noqa: BLE001 -- reported below
            errors.append(e)

    threads = [threading.Thread(target=work, args=(i,)) for i in range(4)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not errors and not wrong, (errors[:1], wrong[:5])
    assert hk.device_status() == 0
