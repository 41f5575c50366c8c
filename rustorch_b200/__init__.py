"""rustorch_b200 — B200-native (sm_100a) dense-contraction backend for RusTorch.

Host-side mirror of the reference's operator interface for this path, over the
C ABI in include/rustorch_b200.h:

    ops.matmul(lhs, rhs)                         rustorch-core/src/ops.rs:1888
    ops.matmul_fused(lhs, rhs, bias, activation) rustorch-core/src/ops.rs:1543
    ops.conv2d(input, weight, stride, padding)   rustorch-core/src/ops/conv.rs:738
    nn.Linear / nn.Conv2d                        rustorch-nn/src/{linear,conv}.rs
    jit.Graph / NodeType / Optimizer / Executor  rustorch-core/src/jit.rs

Tensors are torch CUDA float32 tensors (torch provides device memory and
streams only; all arithmetic runs in this library's kernels).  Calls are
ordered on torch's current stream of the tensor's device.
"""
from __future__ import annotations

import ctypes
import threading

from . import _lib
from ._lib import (ACT_NONE, ACT_RELU, ACT_SIGMOID, ACT_TANH, LAYOUT_NCHW, LAYOUT_NHWC,
                   PREC_3XTF32, PREC_DEFAULT, PREC_TF32, RtbError, call, lib)

__all__ = ["Context", "get_context", "sgemm", "sgemm_batched", "matmul_bias_norm_activation",
           "layer_norm",
           "conv2d_fwd", "matmul_backward",
           "conv2d_backward", "layer_norm_fwd", "layer_norm_backward", "fp8_quantize",
           "fp8_dequantize", "fp8_matmul", "matmul_backward_fp8", "max_pool2d",
           "global_avg_pool", "add", "relu", "fill_normal", "fill_uniform", "RtbError",
           "ACT_NONE", "ACT_RELU", "ACT_SIGMOID", "ACT_TANH", "PREC_3XTF32", "PREC_TF32",
           "PREC_DEFAULT", "LAYOUT_NCHW", "LAYOUT_NHWC", "lib"]


class Context:
    """An rtb_ctx on one device (stream, error word, workspace pool)."""

    def __init__(self, device: int = 0):
        self.device = device
        h = ctypes.c_void_p()
        call("rtb_init", device, ctypes.byref(h))
        self.handle = h

    def close(self) -> None:
        if self.handle:
            call("rtb_destroy", self.handle)
            self.handle = None

    def info(self):
        sm, ma, mi = ctypes.c_int(), ctypes.c_int(), ctypes.c_int()
        mem = ctypes.c_size_t()
        call("rtb_get_device_info", self.handle, ctypes.byref(sm), ctypes.byref(ma),
             ctypes.byref(mi), ctypes.byref(mem))
        return {"sm_count": sm.value, "cc": (ma.value, mi.value), "total_mem": mem.value}

    def set_timeout_ns(self, ns: int) -> None:
        call("rtb_set_timeout_ns", self.handle, int(ns))

    def device_error(self) -> int:
        """Synchronise and read/clear the device error word (0 = none)."""
        code = ctypes.c_int()
        st = lib().rtb_device_error(self.handle, ctypes.byref(code))
        if st not in (_lib.RTB_OK, _lib.RTB_E_TIMEOUT):
            _lib.check(st, "rtb_device_error")
        return code.value

    def synchronize(self, stream=None) -> None:
        call("rtb_stream_synchronize", self.handle, stream)


_ctx_lock = threading.Lock()
_contexts: dict = {}


def get_context(device: int = 0) -> Context:
    c = _contexts.get(device)
    if c is None:
        with _ctx_lock:
            c = _contexts.get(device)
            if c is None:
                c = Context(device)
                _contexts[device] = c
    return c


def _torch():
    import torch
    return torch


def _stream_of(t):
    # the raw handle (an int): making a torch Stream object for it costs 2 us a
    # call, a tenth of a small operator's time
    return _torch()._C._cuda_getCurrentRawStream(t.get_device())


def _dev(t) -> int:
    return t.device.index if t.device.index is not None else 0


def _check_f32_cuda(*ts):
    f32 = _torch().float32
    for t in ts:
        if t is not None and not (t.is_cuda and t.dtype is f32):
            raise ValueError("rustorch_b200 expects float32 CUDA tensors")


def _ptr(t):
    return t.data_ptr() if t is not None else None


def _operand_2d(t):
    """(tensor, leading dim, trans) for a 2-D strided view without copying when
    one dimension is unit-stride; trans=1 means stored as the transpose."""
    if t.stride(1) == 1 and t.stride(0) >= max(t.shape[1], 1):
        return t, t.stride(0), 0
    if t.stride(0) == 1 and t.stride(1) >= max(t.shape[0], 1):
        return t, t.stride(1), 1
    t = t.contiguous()
    return t, t.shape[1], 0


def sgemm(a, b, bias=None, act: int = ACT_NONE, precision: int = PREC_DEFAULT, out=None):
    """C = act(a @ b + bias) for 2-D float32 CUDA tensors a [M,K], b [K,N]."""
    torch = _torch()
    _check_f32_cuda(a, b, bias, out)
    if a.dim() != 2 or b.dim() != 2:
        raise ValueError("Matmul only supports 2D")
    M, K = a.shape
    K2, N = b.shape
    if K != K2:
        raise ValueError("Matmul dimension mismatch")
    if out is None:
        out = torch.empty((M, N), dtype=torch.float32, device=a.device)
    a_, lda, ta = _operand_2d(a)
    b_, ldb, tb = _operand_2d(b)
    if bias is not None:
        bias = bias.contiguous()
    ctx = get_context(_dev(a))
    call("rtb_sgemm", ctx.handle, M, N, K, _ptr(a_), lda, ta, _ptr(b_), ldb, tb, _ptr(bias), act,
         _ptr(out), out.stride(0), precision, _stream_of(a))
    return out


def matmul_bias_norm_activation(a, b, bias=None, norm_weight=None, norm_bias=None,
                                eps: float = 1e-5, act: int = ACT_NONE,
                                precision: int = PREC_DEFAULT, out=None):
    """ops::matmul_bias_norm_activation: act(layer_norm(a @ b + bias) * norm_weight
    + norm_bias), the LayerNorm over the last dimension (N), for 2-D float32
    CUDA tensors a [M,K], b [K,N]; act is any ACT_*."""
    torch = _torch()
    _check_f32_cuda(a, b, bias, norm_weight, norm_bias, out)
    if a.dim() != 2 or b.dim() != 2:
        raise ValueError("Matmul only supports 2D")
    M, K = a.shape
    K2, N = b.shape
    if K != K2:
        raise ValueError("Matmul dimension mismatch")
    for t in (bias, norm_weight, norm_bias):
        if t is not None and t.numel() != N:
            raise ValueError("bias / norm parameters must have N elements")
    if out is None:
        out = torch.empty((M, N), dtype=torch.float32, device=a.device)
    a_, lda, ta = _operand_2d(a)
    b_, ldb, tb = _operand_2d(b)
    bias, norm_weight, norm_bias = (t.contiguous() if t is not None else None
                                    for t in (bias, norm_weight, norm_bias))
    ctx = get_context(_dev(a))
    call("rtb_matmul_bias_norm_act", ctx.handle, M, N, K, _ptr(a_), lda, ta, _ptr(b_), ldb, tb,
         _ptr(bias), _ptr(norm_weight), _ptr(norm_bias), float(eps), act, _ptr(out),
         out.stride(0), precision, _stream_of(a))
    return out


def layer_norm(x, norm_weight=None, norm_bias=None, eps: float = 1e-5, act: int = ACT_NONE,
               out=None):
    """ops::layer_norm over the last dimension (+ an optional activation) for a
    float32 CUDA tensor whose rows are contiguous; out may be x (in place)."""
    torch = _torch()
    _check_f32_cuda(x, norm_weight, norm_bias, out)
    if x.dim() == 0:
        raise ValueError("LayerNorm: Input shape smaller than normalized shape")
    d = x.shape[-1]
    x2 = _rows_2d(x, d) if d else x.reshape(-1, 0)
    for t in (norm_weight, norm_bias):
        if t is not None and t.numel() != d:
            raise ValueError("LayerNorm: Input shape does not match normalized shape")
    if out is None:
        out = torch.empty(x.shape, dtype=torch.float32, device=x.device)
    y2 = out.view(-1, d) if d else out.reshape(-1, 0)
    norm_weight, norm_bias = (t.contiguous() if t is not None else None
                              for t in (norm_weight, norm_bias))
    ctx = get_context(_dev(x))
    call("rtb_layer_norm", ctx.handle, x2.shape[0], d, _ptr(x2), max(x2.stride(0), d),
         _ptr(norm_weight), _ptr(norm_bias), float(eps), act, _ptr(y2), max(y2.stride(0), d),
         _stream_of(x))
    return out


def sgemm_batched(a, b, bias=None, act: int = ACT_NONE, precision: int = PREC_DEFAULT):
    """Batched C[i] = act(a[i] @ b[i] + bias) for contiguous 3-D tensors."""
    torch = _torch()
    _check_f32_cuda(a, b, bias)
    a = a.contiguous()
    b = b.contiguous()
    Bt, M, K = a.shape
    _, K2, N = b.shape
    if K != K2 or b.shape[0] != Bt:
        raise ValueError("batched matmul dimension mismatch")
    out = torch.empty((Bt, M, N), dtype=torch.float32, device=a.device)
    ctx = get_context(_dev(a))
    call("rtb_sgemm_batched", ctx.handle, Bt, M, N, K, _ptr(a), K, M * K, 0, _ptr(b), N, K * N, 0,
         _ptr(bias.contiguous() if bias is not None else None), act, _ptr(out), N, M * N,
         precision, _stream_of(a))
    return out


def conv_out_hw(h, w, kh, kw, stride, padding):
    return (h + 2 * padding[0] - kh) // stride[0] + 1, (w + 2 * padding[1] - kw) // stride[1] + 1


def conv2d_fwd(x, w, bias=None, stride=(1, 1), padding=(0, 0), residual=None, act: int = ACT_NONE,
               x_layout: int = LAYOUT_NCHW, y_layout: int = LAYOUT_NCHW,
               precision: int = PREC_DEFAULT):
    """y = act(conv2d(x, w) + bias + residual); w is [Co, Ci, kh, kw]."""
    torch = _torch()
    _check_f32_cuda(x, w, bias, residual)
    x = x.contiguous()
    w = w.contiguous()
    if x_layout == LAYOUT_NCHW:
        N, Ci, H, W = x.shape
    else:
        N, H, W, Ci = x.shape
    Co, Ci2, kh, kw = w.shape
    if Ci2 != Ci:
        raise ValueError(f"Weight input channels {Ci2} must match input channels {Ci}")
    Ho, Wo = conv_out_hw(H, W, kh, kw, stride, padding)
    shape = (N, Co, Ho, Wo) if y_layout == LAYOUT_NCHW else (N, Ho, Wo, Co)
    y = torch.empty(shape, dtype=torch.float32, device=x.device)
    if residual is not None:
        residual = residual.contiguous()
    ctx = get_context(_dev(x))
    call("rtb_conv2d_fwd", ctx.handle, N, Ci, H, W, Co, kh, kw, stride[0], stride[1], padding[0],
         padding[1], _ptr(x), x_layout, _ptr(w), _ptr(bias.contiguous() if bias is not None else None),
         _ptr(residual), act, _ptr(y), y_layout, precision, _stream_of(x))
    return y


def matmul_backward(a, b, grad, need_a: bool = True, need_b: bool = True, out_a=None, out_b=None,
                    accumulate: bool = False, precision: int = PREC_DEFAULT):
    """MatmulBackward of c = a @ b: (grad @ b.T, a.T @ grad) for contiguous 2-D
    float32 CUDA tensors; with accumulate the results are added to out_a/out_b."""
    torch = _torch()
    _check_f32_cuda(a, b, grad)
    a, b, grad = a.contiguous(), b.contiguous(), grad.contiguous()
    M, K = a.shape
    N = b.shape[1]
    if b.shape[0] != K or tuple(grad.shape) != (M, N):
        raise ValueError("matmul_backward: shape mismatch")
    da = (out_a if out_a is not None else torch.empty((M, K), dtype=torch.float32,
                                                      device=a.device)) if need_a else None
    db = (out_b if out_b is not None else torch.empty((K, N), dtype=torch.float32,
                                                      device=a.device)) if need_b else None
    ctx = get_context(_dev(a))
    call("rtb_matmul_backward", ctx.handle, M, N, K, _ptr(a), _ptr(b), _ptr(grad), _ptr(da),
         _ptr(db), int(accumulate), precision, _stream_of(a))
    return da, db


def conv2d_backward(x, w, grad, stride=(1, 1), padding=(0, 0), need_x: bool = True,
                    need_w: bool = True, precision: int = PREC_DEFAULT):
    """Conv2dBackward (NCHW): (grad wrt x, grad wrt w) of y = conv2d(x, w)."""
    torch = _torch()
    _check_f32_cuda(x, w, grad)
    x, w, grad = x.contiguous(), w.contiguous(), grad.contiguous()
    N, Ci, H, W = x.shape
    Co, _, kh, kw = w.shape
    dx = torch.empty_like(x) if need_x else None
    dw = torch.empty_like(w) if need_w else None
    ctx = get_context(_dev(x))
    call("rtb_conv2d_backward", ctx.handle, N, Ci, H, W, Co, kh, kw, stride[0], stride[1],
         padding[0], padding[1], _ptr(x), _ptr(w), _ptr(grad), _ptr(dx), _ptr(dw), 0, precision,
         _stream_of(x))
    return dx, dw


def _rows_2d(t, d):
    """t as [rows, d] with contiguous rows that do not overlap (a copy only where
    t has no such view: a transposed or an expanded tensor)."""
    if t.is_contiguous():
        return t if t.dim() == 2 else t.view(-1, d)
    t2 = t.reshape(-1, d) if t.dim() != 2 else t
    if (d > 1 and t2.stride(1) != 1) or (t2.shape[0] > 1 and t2.stride(0) < d):
        t2 = t2.contiguous()
    return t2


def _ld(t, d):
    """Leading dimension of _rows_2d's result (a single row's stride says nothing)."""
    return max(t.stride(0), d)


def _flat(t, n, message):
    """A vector of n elements, contiguous; None stays None."""
    if t is None:
        return None
    if t.numel() != n:
        raise ValueError(message)
    return t if t.is_contiguous() else t.contiguous()


def _same_device(first, *rest):
    dev = first.get_device()
    for t in rest:
        if t is not None and t.get_device() != dev:
            raise ValueError("rustorch_b200: tensors on different devices")
    return dev


def _empty_like(x):
    """float32, contiguous, of x's shape and on its device."""
    torch = _torch()
    if x.dtype is torch.float32 and x.is_contiguous():
        return torch.empty_like(x)
    return torch.empty(x.shape, dtype=torch.float32, device=x.device)


def _result(out, need, accumulate, shape, like, who):
    """The tensor that a gradient is written to (or added to): `out` or a new one."""
    if not need:
        return None
    if out is None:
        if accumulate:
            raise ValueError(f"{who}: accumulate adds to given outputs")
        return like.new_empty(shape, dtype=_torch().float32)
    if not out.is_contiguous() or tuple(out.shape) != tuple(shape):
        raise ValueError(f"{who}: outputs must be contiguous and of the gradient's shape")
    return out


_LN_SHAPE = "LayerNorm: Input shape does not match normalized shape"


def layer_norm_fwd(x, norm_weight=None, norm_bias=None, eps: float = 1e-5, act: int = ACT_NONE,
                   out=None):
    """layer_norm that also returns what its backward pass reads: (y, mean,
    rstd), the statistics float32 of x's leading shape; out may be x."""
    _check_f32_cuda(x, norm_weight, norm_bias, out)
    dev = _same_device(x, norm_weight, norm_bias, out)
    d = x.shape[-1] if x.dim() else 0
    if d == 0:
        raise ValueError("LayerNorm: Input shape smaller than normalized shape")
    w, b = _flat(norm_weight, d, _LN_SHAPE), _flat(norm_bias, d, _LN_SHAPE)
    x2 = _rows_2d(x, d)
    if out is None:
        out = y2 = _empty_like(x)
        ldy = d
    else:
        if out.shape != x.shape or (d > 1 and out.stride(-1) != 1):
            raise ValueError("layer_norm_fwd: out must have x's shape and contiguous rows")
        y2 = out if out.dim() == 2 else out.view(-1, d)
        if y2.shape[0] > 1 and y2.stride(0) < d:
            raise ValueError("layer_norm_fwd: out's rows overlap")
        ldy = _ld(y2, d)
    mean = x.new_empty(x.shape[:-1])
    rstd = x.new_empty(x.shape[:-1])
    call("rtb_layer_norm_fwd", get_context(dev).handle, x2.shape[0], d, _ptr(x2), _ld(x2, d),
         _ptr(w), _ptr(b), eps, act, _ptr(y2), ldy, _ptr(mean), _ptr(rstd), _stream_of(x))
    return out, mean, rstd


def layer_norm_backward(x, mean, rstd, grad, norm_weight=None, norm_bias=None,
                        act: int = ACT_NONE, x_scale=None, need_x: bool = True,
                        need_weight: bool = True, need_bias: bool = True, out_x=None,
                        out_weight=None, out_bias=None, accumulate: bool = False):
    """Gradients (dx, dweight, dbias) of layer_norm_fwd for the incoming
    gradient `grad`; x is the forward's input, float32 or an 8-bit checkpoint
    (fp8_quantize(x) -> x, x_scale).  With accumulate the results are added to
    out_x / out_weight / out_bias."""
    who = "layer_norm_backward"
    saved = x.dtype is _torch().float8_e4m3fn
    _check_f32_cuda(mean, rstd, grad, norm_weight, norm_bias, out_x, out_weight, out_bias)
    if not saved:
        _check_f32_cuda(x)
    dev = _same_device(x, mean, rstd, grad, norm_weight, norm_bias, x_scale, out_x, out_weight,
                       out_bias)
    d = x.shape[-1] if x.dim() else 0
    if d == 0 or grad.shape != x.shape:
        raise ValueError("layer_norm_backward: grad must have x's shape, with a last dimension")
    x2, g2 = _rows_2d(x, d), _rows_2d(grad, d)
    rows = x2.shape[0]
    per_row = "layer_norm_backward: one mean and rstd for each row"
    mean, rstd = _flat(mean, rows, per_row), _flat(rstd, rows, per_row)
    w, b = _flat(norm_weight, d, _LN_SHAPE), _flat(norm_bias, d, _LN_SHAPE)
    if saved != (x_scale is not None):
        raise ValueError("layer_norm_backward: x_scale goes with an 8-bit x, and only with one")
    dx = _result(out_x, need_x, accumulate, x.shape, grad, who)
    dw = _result(out_weight, need_weight, accumulate, (d,), grad, who)
    db = _result(out_bias, need_bias, accumulate, (d,), grad, who)
    rest = (_ptr(mean), _ptr(rstd), _ptr(w), _ptr(b), act, _ptr(g2), _ld(g2, d), _ptr(dx), d,
            _ptr(dw), _ptr(db), bool(accumulate), _stream_of(x))
    h = get_context(dev).handle
    if saved:
        s2, block_rows, kind = _scales(x_scale, rows, d, who)
        if kind != _lib.SCALE_E8M0 or block_rows != 1:
            raise ValueError("layer_norm_backward: a checkpoint has a power-of-two scale for each "
                             "128 columns of a row")
        call("rtb_layer_norm_backward_fp8", h, rows, d, _ptr(x2), _ld(x2, d), _ptr(s2),
             _ld(s2, s2.shape[1]), *rest)
    else:
        call("rtb_layer_norm_backward", h, rows, d, _ptr(x2), _ld(x2, d), *rest)
    return dx, dw, db


def _scales(scale, rows, cols, who):
    """(2-D scales with contiguous rows, block_rows, scale type) of a [rows, cols] 8-bit tensor."""
    torch = _torch()
    e8m0 = scale.dtype is torch.float8_e8m0fnu
    if not scale.is_cuda or not (e8m0 or scale.dtype is torch.float32):
        raise ValueError(f"{who}: scales are float8_e8m0fnu or float32 CUDA tensors")
    cb = (cols + 127) // 128
    s = _rows_2d(scale, cb)
    n = s.shape[0]
    if s.shape[1] != cb or n not in (rows, (rows + 127) // 128):
        raise ValueError(f"{who}: scales must be [rows or ceil(rows / 128), ceil(cols / 128)]")
    return s, 1 if n == rows else 128, _lib.SCALE_E8M0 if e8m0 else _lib.SCALE_F32


def _check_fp8(who, *ts):
    e4m3 = _torch().float8_e4m3fn
    for t in ts:
        if not (t.is_cuda and t.dtype is e4m3):
            raise ValueError(f"{who} expects float8_e4m3fn CUDA tensors")


def fp8_quantize(x, block_rows: int = 1):
    """(q, scale): x [..., cols] as e4m3 values with one power-of-two scale
    (float8_e8m0fnu) for each 128 columns of a row (block_rows = 1) or of 128
    rows of a 2-D x (block_rows = 128).  An activation checkpoint, and an
    operand of fp8_matmul."""
    torch = _torch()
    _check_f32_cuda(x)
    if block_rows not in (1, 128):
        raise ValueError("fp8_quantize: block_rows must be 1 or 128")
    if x.dim() == 0 or (block_rows != 1 and x.dim() != 2):
        raise ValueError("fp8_quantize: x needs a last dimension, and two for 128-row blocks")
    cols = x.shape[-1]
    cb = (cols + 127) // 128
    q = x.new_empty(x.shape, dtype=torch.float8_e4m3fn)
    lead = x.shape[:-1] if block_rows == 1 else ((x.shape[0] + 127) // 128,)
    scale = x.new_empty((*lead, cb), dtype=torch.float8_e8m0fnu)
    if x.numel():
        x2 = _rows_2d(x, cols)
        call("rtb_fp8_quantize", get_context(x.get_device()).handle, x2.shape[0], cols, _ptr(x2),
             _ld(x2, cols), block_rows, _ptr(q), cols, _ptr(scale), cb, _stream_of(x))
    return q, scale


def fp8_dequantize(q, scale, out=None):
    """The float32 values q * scale of fp8_quantize's (q, scale)."""
    _check_fp8("fp8_dequantize", q)
    _check_f32_cuda(out)
    dev = _same_device(q, scale, out)
    if q.dim() == 0:
        raise ValueError("fp8_dequantize: q needs a last dimension")
    cols = q.shape[-1]
    if out is None:
        out = _empty_like(q)
    elif out.shape != q.shape or not out.is_contiguous():
        raise ValueError("fp8_dequantize: out must be contiguous and have q's shape")
    if q.numel():
        q2 = _rows_2d(q, cols)
        rows = q2.shape[0]
        s, block_rows, kind = _scales(scale, rows, cols, "fp8_dequantize")
        if kind != _lib.SCALE_E8M0:
            raise ValueError("fp8_dequantize: scales are float8_e8m0fnu")
        call("rtb_fp8_dequantize", get_context(dev).handle, rows, cols, _ptr(q2), _ld(q2, cols),
             _ptr(s), _ld(s, s.shape[1]), block_rows, _ptr(out), cols, _stream_of(q))
    return out


def fp8_matmul(a, a_scale, b, b_scale, bias=None, act: int = ACT_NONE, out=None):
    """C = act(deq(a) @ deq(b) + bias), float32, for block-scaled 8-bit a [M,K]
    and b [K,N].  b is a Linear weight's transposed view (w.t(), with its
    scales' ws.t()) or a row-major matrix with 128 x 128 blocks; scales are
    float8_e8m0fnu or float32."""
    _check_fp8("fp8_matmul", a, b)
    _check_f32_cuda(bias, out)
    dev = _same_device(a, a_scale, b, b_scale, bias, out)
    if a.dim() != 2 or b.dim() != 2 or b_scale.dim() != 2:
        raise ValueError("Matmul only supports 2D")
    M, K = a.shape
    K2, N = b.shape
    if K != K2:
        raise ValueError("Matmul dimension mismatch")
    bias = _flat(bias, N, "fp8_matmul: bias must have N elements")
    if out is None:
        out = a.new_empty((M, N), dtype=_torch().float32)
    elif tuple(out.shape) != (M, N) or (N > 1 and out.stride(1) != 1) or (
            M > 1 and out.stride(0) < N):
        raise ValueError("fp8_matmul: out must be [M, N] with contiguous rows")
    a_ = _rows_2d(a, K)
    sa, ra, ka = _scales(a_scale, M, K, "fp8_matmul")
    if b.stride(0) == 1 or b.stride(1) != 1:
        w, trans = _rows_2d(b.t(), K), 1
        sb, rb_, kb = _scales(b_scale.t(), N, K, "fp8_matmul")
    else:
        w, trans = _rows_2d(b, N), 0
        sb, rb_, kb = _scales(b_scale, K, N, "fp8_matmul")
        if rb_ != 128 and K > 1:
            raise ValueError("fp8_matmul: a row-major b needs 128 x 128 blocks")
        rb_ = 128
    call("rtb_fp8_matmul", get_context(dev).handle, M, N, K, _ptr(a_), _ld(a_, K), _ptr(sa),
         _ld(sa, sa.shape[1]), ra, ka, _ptr(w), _ld(w, w.shape[1]), trans, _ptr(sb),
         _ld(sb, sb.shape[1]), rb_, kb, _ptr(bias), act, _ptr(out), _ld(out, N), _stream_of(a))
    return out


def matmul_backward_fp8(a, a_scale, b, grad, need_a: bool = True, need_b: bool = True, out_a=None,
                        out_b=None, accumulate: bool = False, precision: int = PREC_DEFAULT):
    """matmul_backward of c = a @ b with a [M,K] kept as an 8-bit checkpoint
    (fp8_quantize): (grad @ b.T, deq(a).T @ grad); b (float32 [K,N]) is read for
    the first only and may be None without it.  With accumulate the results
    are added to out_a / out_b."""
    who = "matmul_backward_fp8"
    _check_fp8(who, a)
    _check_f32_cuda(b, grad, out_a, out_b)
    dev = _same_device(a, a_scale, b, grad, out_a, out_b)
    if a.dim() != 2 or grad.dim() != 2:
        raise ValueError("Matmul only supports 2D")
    M, K = a.shape
    N = grad.shape[1]
    if grad.shape[0] != M or (b is not None and tuple(b.shape) != (K, N)):
        raise ValueError("matmul_backward_fp8: shape mismatch")
    if need_a and b is None:
        raise ValueError("matmul_backward_fp8: the gradient of a needs b")
    da = _result(out_a, need_a, accumulate, (M, K), grad, who)
    db = _result(out_b, need_b, accumulate, (K, N), grad, who)
    if not grad.is_contiguous():
        grad = grad.contiguous()
    b = b.contiguous() if b is not None and need_a else None
    a_ = _rows_2d(a, K)
    sa, ra, kind = _scales(a_scale, M, K, who)
    if kind != _lib.SCALE_E8M0:
        raise ValueError("matmul_backward_fp8: a checkpoint's scales are float8_e8m0fnu")
    call("rtb_matmul_backward_fp8", get_context(dev).handle, M, N, K, _ptr(a_), _ld(a_, K),
         _ptr(sa), _ld(sa, sa.shape[1]), ra, _ptr(b), _ptr(grad), _ptr(da), _ptr(db),
         bool(accumulate), precision, _stream_of(a))
    return da, db


def max_pool2d(x, kernel=(3, 3), stride=(2, 2), padding=(1, 1), layout: int = LAYOUT_NCHW):
    torch = _torch()
    _check_f32_cuda(x)
    x = x.contiguous()
    if layout == LAYOUT_NCHW:
        N, C, H, W = x.shape
    else:
        N, H, W, C = x.shape
    Ho, Wo = conv_out_hw(H, W, kernel[0], kernel[1], stride, padding)
    shape = (N, C, Ho, Wo) if layout == LAYOUT_NCHW else (N, Ho, Wo, C)
    y = torch.empty(shape, dtype=torch.float32, device=x.device)
    ctx = get_context(_dev(x))
    call("rtb_max_pool2d", ctx.handle, N, C, H, W, kernel[0], kernel[1], stride[0], stride[1],
         padding[0], padding[1], _ptr(x), _ptr(y), layout, _stream_of(x))
    return y


def global_avg_pool(x, layout: int = LAYOUT_NCHW):
    torch = _torch()
    _check_f32_cuda(x)
    x = x.contiguous()
    if layout == LAYOUT_NCHW:
        N, C, H, W = x.shape
    else:
        N, H, W, C = x.shape
    y = torch.empty((N, C), dtype=torch.float32, device=x.device)
    ctx = get_context(_dev(x))
    call("rtb_global_avg_pool", ctx.handle, N, C, H, W, _ptr(x), _ptr(y), layout, _stream_of(x))
    return y


def add(a, b):
    torch = _torch()
    _check_f32_cuda(a, b)
    if a.shape != b.shape:
        raise ValueError("add: shapes differ")
    a = a.contiguous()
    b = b.contiguous()
    y = torch.empty_like(a)
    call("rtb_add", get_context(_dev(a)).handle, a.numel(), _ptr(a), _ptr(b), _ptr(y),
         _stream_of(a))
    return y


def relu(x):
    torch = _torch()
    _check_f32_cuda(x)
    x = x.contiguous()
    y = torch.empty_like(x)
    call("rtb_relu", get_context(_dev(x)).handle, x.numel(), _ptr(x), _ptr(y), _stream_of(x))
    return y


def fill_normal(shape, seed: int, tensor_id: int, mean: float = 0.0, std: float = 1.0):
    """Host numpy array from the documented SplitMix64/Box-Muller generator."""
    import numpy as np
    out = np.empty(shape, dtype=np.float32)
    call("rtb_fill_normal_host", out.ctypes.data_as(ctypes.c_void_p), out.size, seed, tensor_id,
         mean, std)
    return out


def fill_uniform(shape, seed: int, tensor_id: int, lo: float, hi: float):
    import numpy as np
    out = np.empty(shape, dtype=np.float32)
    call("rtb_fill_uniform_host", out.ctypes.data_as(ctypes.c_void_p), out.size, seed, tensor_id,
         lo, hi)
    return out
