"""Refusals of the root-mean-square norm's and the 4-bit entry points that need no GPU:
a null context, bad sizes and pointers (no device is touched: the context is a block of
zeros), tensors that are not on a GPU, whole numbers out of range."""
import ctypes
import os

import pytest
import torch


@pytest.fixture(scope="module")
def rb():
    from rustorch_b200 import build
    build.build()
    import rustorch_b200
    rustorch_b200.lib()
    return rustorch_b200


P = ctypes.c_void_p(1 << 20)
Q = ctypes.c_void_p(1 << 24)


def entries(L):
    """name -> (call, good arguments by name): rows or M 2, columns or K 64, N 3."""
    norm = dict(rows=2, d=64, x=P, ldx=64, residual=None, ldr=0, weight=None, eps=1e-5, sum=None, ldsum=0)
    back = dict(rstd=P, weight=None, dy=P, lddy=64, dsum=None, ldds=0, dx=Q, lddx=64, dw=None, accumulate=0)
    return {
        "rtb_rms_norm_fwd": {**norm, "y": Q, "ldy": 64, "rstd": P},
        "rtb_rms_norm_fp8": {**norm, "q": Q, "ldq": 64, "scale": Q, "lds": 1, "rstd": P},
        "rtb_rms_norm_backward": {"rows": 2, "d": 64, "x": P, "ldx": 64, **back},
        "rtb_rms_norm_backward_fp8": {"rows": 2, "d": 64, "q": P, "ldq": 64, "scale": P, "lds": 1, **back},
        "rtb_fp4_quantize": dict(rows=2, cols=64, x=P, ldx=64, trans=0, q=Q, ldq=32, scale=Q, lds=2),
        "rtb_fp4_dequantize": dict(rows=2, cols=64, q=P, ldq=32, scale=P, lds=2, y=Q, ldy=64),
        "rtb_fp4_matmul": dict(M=2, N=3, K=64, a=P, lda=32, sa=P, ldsa=2, b=P, ldb=32, sb=P, ldsb=2, bias=None, act=0, c=Q,
                               ldc=3),
    }


def test_null_context(rb):
    for name, args in entries(rb.lib()).items():
        assert getattr(rb.lib(), name)(None, *args.values(), None) == rb._lib.RTB_E_INVALID
        assert "rtb_ctx" in rb._lib.last_error()


BAD = [("rtb_rms_norm_fwd", bad) for bad in
       (dict(rows=-1), dict(d=-1), dict(d=0), dict(x=None), dict(y=None), dict(ldx=63), dict(ldy=63),
        dict(residual=P, ldr=63), dict(sum=Q, ldsum=63), dict(sum=Q, ldsum=64))]
BAD += [("rtb_rms_norm_fp8", bad) for bad in
        (dict(rows=-1), dict(d=-1), dict(d=0), dict(x=None), dict(q=None), dict(scale=None), dict(ldx=63), dict(ldq=63),
         dict(lds=0), dict(residual=P, ldr=63), dict(sum=P, ldsum=63))]
BAD += [("rtb_rms_norm_backward", bad) for bad in
        (dict(rows=-1), dict(d=-1), dict(x=None), dict(rstd=None), dict(dy=None), dict(ldx=63), dict(lddy=63),
         dict(dsum=P, ldds=63), dict(lddx=63))]
BAD += [("rtb_rms_norm_backward_fp8", bad) for bad in
        (dict(rows=-1), dict(d=-1), dict(q=None), dict(scale=None), dict(ldq=63), dict(lds=0), dict(rstd=None),
         dict(dy=None), dict(dsum=P, ldds=63), dict(lddx=63))]
BAD += [("rtb_fp4_quantize", bad) for bad in
        (dict(rows=-1), dict(cols=-1), dict(x=None), dict(q=None), dict(scale=None), dict(ldx=63), dict(ldq=31), dict(lds=1),
         dict(trans=2), dict(trans=1, ldx=1), dict(cols=65))]
BAD += [("rtb_fp4_dequantize", bad) for bad in
        (dict(rows=-1), dict(cols=-1), dict(q=None), dict(scale=None), dict(y=None), dict(ldq=31), dict(lds=1), dict(ldy=63),
         dict(cols=65))]
BAD += [("rtb_fp4_matmul", bad) for bad in
        (dict(M=-1), dict(N=-1), dict(K=-2), dict(K=63), dict(act=4), dict(act=-1), dict(a=None), dict(b=None), dict(sa=None),
         dict(sb=None), dict(c=None), dict(lda=31), dict(ldb=31), dict(ldsa=1), dict(ldsb=1), dict(ldc=2), dict(N=4))]


@pytest.mark.parametrize("name,bad", BAD)
def test_bad_arguments(rb, name, bad):
    if torch.cuda.is_available():
        pytest.skip("checked where nothing can be launched")
    ctx = ctypes.create_string_buffer(4096)
    args = {**entries(rb.lib())[name], **bad}
    assert getattr(rb.lib(), name)(ctx, *args.values(), None) == rb._lib.RTB_E_INVALID, rb._lib.last_error()


@pytest.mark.parametrize("name,big", [("rtb_rms_norm_fwd", dict(d=2 ** 31 - 1, ldx=2 ** 31, ldy=2 ** 31)),
                                      ("rtb_rms_norm_fp8", dict(d=2 ** 31 - 1, ldx=2 ** 31, ldq=2 ** 31, lds=2 ** 25)),
                                      ("rtb_rms_norm_backward", dict(d=2 ** 31 - 1, ldx=2 ** 31, lddy=2 ** 31, lddx=2 ** 31)),
                                      ("rtb_fp4_quantize", dict(cols=2 ** 31, ldx=2 ** 31, ldq=2 ** 30, lds=2 ** 26)),
                                      ("rtb_fp4_dequantize", dict(cols=2 ** 31, ldy=2 ** 31, ldq=2 ** 30, lds=2 ** 26)),
                                      ("rtb_fp4_matmul", dict(M=2 ** 31)),
                                      ("rtb_fp4_matmul", dict(N=2 ** 31, ldc=2 ** 31)),
                                      ("rtb_fp4_matmul", dict(K=2 ** 31, lda=2 ** 30, ldb=2 ** 30, ldsa=2 ** 26, ldsb=2 ** 26))])
def test_sizes_beyond_the_index_range_refused(rb, name, big):
    if torch.cuda.is_available():
        pytest.skip("checked where nothing can be launched")
    ctx = ctypes.create_string_buffer(4096)
    args = {**entries(rb.lib())[name], **big}
    assert getattr(rb.lib(), name)(ctx, *args.values(), None) == rb._lib.RTB_E_UNSUPPORTED, rb._lib.last_error()


def host_calls(rb):
    x, m = torch.zeros((4, 128)), torch.zeros(4)
    q = torch.zeros((4, 64), dtype=torch.uint8).view(torch.float4_e2m1fn_x2)
    s = torch.full((4, 4), 127, dtype=torch.uint8).view(torch.float8_e8m0fnu)
    return (lambda: rb.rms_norm_fwd(x), lambda: rb.rms_norm_fp8(x), lambda: rb.rms_norm_backward(x, m, x),
            lambda: rb.rms_norm_backward(x.to(torch.float8_e4m3fn), m, x, x_scale=s[:, :1]), lambda: rb.fp4_quantize(x),
            lambda: rb.fp4_dequantize(q, s), lambda: rb.fp4_matmul(q, s, q.t(), s.t()),
            lambda: rb.fp4_matmul(q, s, q.t(), s.t(), act=2 ** 32), lambda: rb.fp4_dequantize(q, s, 2 ** 32 + 128))


@pytest.mark.parametrize("k", range(9))
def test_host_tensors_and_whole_numbers_refused(rb, k):
    with pytest.raises(ValueError):
        host_calls(rb)[k]()


def test_no_tensor_refused(rb):
    for call in (lambda: rb.rms_norm_fwd(None), lambda: rb.fp4_quantize([1.0]), lambda: rb.fp4_matmul(1, 2, 3, 4)):
        with pytest.raises(TypeError):
            call()


def test_no_hidden_switches():
    """The kernels of these operators are chosen by the call's sizes, types and alignment
    and by nothing in the environment."""
    csrc = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "rustorch_b200", "csrc")
    for name in os.listdir(csrc):
        if name.startswith(("rtb_rms", "rtb_fp4")):
            with open(os.path.join(csrc, name)) as f:
                assert "getenv" not in f.read(), name
