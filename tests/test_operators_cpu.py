"""Refusals of the training and 8-bit entry points that need no GPU: a null
context, tensors that are not on one, wrong types."""
import ctypes
import os
import subprocess

import pytest
import torch


@pytest.fixture(scope="module")
def rb():
    from rustorch_b200 import build
    build.build()
    import rustorch_b200
    rustorch_b200.lib()
    return rustorch_b200


def test_null_context(rb):
    L = rb.lib()
    for st in (
            L.rtb_layer_norm_fwd(None, 2, 2, None, 2, None, None, 1e-5, 0, None, 2, None, None, None),
            L.rtb_layer_norm_backward(None, 2, 2, None, 2, None, None, None, None, 0, None, 2, None,
                                      2, None, None, 0, None),
            L.rtb_layer_norm_backward_fp8(None, 2, 2, None, 2, None, 1, None, None, None, None, 0,
                                          None, 2, None, 2, None, None, 0, None),
            L.rtb_fp8_quantize(None, 2, 2, None, 2, 1, None, 2, None, 1, None),
            L.rtb_fp8_dequantize(None, 2, 2, None, 2, None, 1, 1, None, 2, None),
            L.rtb_fp8_matmul(None, 2, 2, 2, None, 2, None, 1, 1, 0, None, 2, 1, None, 1, 1, 0, None,
                             0, None, 2, None),
            L.rtb_matmul_backward_fp8(None, 2, 2, 2, None, 2, None, 1, 1, None, None, None, None, 0,
                                      0, None)):
        assert st == rb._lib.RTB_E_INVALID
        assert "rtb_ctx" in rb._lib.last_error()


def test_host_tensors_refused(rb):
    x = torch.zeros((4, 128))
    q = x.to(torch.float8_e4m3fn)
    s = torch.full((4, 1), 127, dtype=torch.uint8).view(torch.float8_e8m0fnu)
    m = torch.zeros(4)
    for call in (lambda: rb.fp8_quantize(x), lambda: rb.fp8_dequantize(q, s),
                 lambda: rb.fp8_matmul(q, s, q.t(), s.t()),
                 lambda: rb.matmul_backward_fp8(q, s, None, x, need_a=False),
                 lambda: rb.layer_norm_fwd(x),
                 lambda: rb.layer_norm_backward(x, m, m, x),
                 lambda: rb.layer_norm_backward(q, m, m, x, x_scale=s)):
        with pytest.raises(ValueError):
            call()


def test_rows_beyond_the_index_range_refused(rb):
    """Rows of almost 2^31 columns off the 16-byte boundaries are refused before
    anything is launched (no device is touched: the context is a block of zeros)."""
    if torch.cuda.is_available():
        pytest.skip("checked where nothing can be launched")
    L = rb.lib()
    ctx = ctypes.create_string_buffer(4096)
    p = ctypes.c_void_p(1 << 20)
    for d in (2 ** 31 - 1, 2 ** 31 - 256):
        ld = d | 1
        st = L.rtb_layer_norm_fwd(ctx, 1, d, p, ld, None, None, 1e-5, 0, p, ld, p, p, None)
        assert st == rb._lib.RTB_E_UNSUPPORTED, rb._lib.last_error()
        st = L.rtb_layer_norm(ctx, 1, d, p, ld, None, None, 1e-5, 0, p, ld, None)
        assert st == rb._lib.RTB_E_UNSUPPORTED, rb._lib.last_error()


@pytest.mark.parametrize("value", [2 ** 32, 2 ** 32 + 1, -2 ** 32 + 3, 2 ** 80])
def test_whole_numbers_out_of_range_refused(rb, value):
    """No argument is taken modulo 2^32 (block_rows 2^32 + 1 as 1, act 2^32 as 0)."""
    x = torch.zeros((4, 128))
    q = x.to(torch.float8_e4m3fn)
    s = torch.full((4, 1), 127, dtype=torch.uint8).view(torch.float8_e8m0fnu)
    m = torch.zeros(4)
    for call in (lambda: rb.fp8_quantize(x, value), lambda: rb.layer_norm_fwd(x, act=value),
                 lambda: rb.layer_norm_backward(x, m, m, x, act=value),
                 lambda: rb.fp8_matmul(q, s, q.t(), s.t(), act=value),
                 lambda: rb.matmul_backward_fp8(q, s, None, x, need_a=False, precision=value)):
        with pytest.raises(ValueError, match="out of range"):
            call()


def test_answers_kept_for_each_device(tmp_path):
    """The cache of what a device holds at once (tests/cpp/test_per_device.cpp)."""
    src = os.path.join(os.path.dirname(os.path.abspath(__file__)), "cpp", "test_per_device.cpp")
    exe = str(tmp_path / "per_device")
    r = subprocess.run(["g++", "-std=c++17", "-O1", src, "-o", exe], capture_output=True, text=True)
    assert r.returncode == 0, r.stderr
    r = subprocess.run([exe], capture_output=True, text=True, timeout=60)
    assert r.returncode == 0 and r.stdout == "fine\n", r.stdout


def test_no_hidden_switches():
    """The kernels of these operators are chosen by the call's sizes and types and by
    nothing in the environment."""
    csrc = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "rustorch_b200", "csrc")
    for name in ("rtb_blockgemm.cu", "rtb_pairgemm.cu", "rtb_mxgemm.cu", "rtb_fp8.cu", "rtb_norm.cu",
                 "rtb_norm_bwd.cu", os.path.join("python", "ops_module.cpp")):
        with open(os.path.join(csrc, name)) as f:
            assert "getenv" not in f.read(), name
