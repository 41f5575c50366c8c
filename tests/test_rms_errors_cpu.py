"""What the root-mean-square norm's entry points refuse, and how they report what failed,
without a GPU: a backward pass that cannot be launched says which one it is (every launch
fails here, on the host); an output in an input's place has to have its rows there too."""
import ctypes

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


# the row kernels, the one of wide rows, the one of any width
@pytest.mark.parametrize("d", [64, 1001, 4096, 8192, 9000, 20000])
def test_launch_errors_name_the_entry_point(rb, d):
    if torch.cuda.is_available():
        pytest.skip("checked where nothing can be launched")
    L = rb.lib()
    blocks = -(-d // 128)
    calls = {
        "layer_norm_backward": lambda ctx: L.rtb_layer_norm_backward(
            ctx, 2, d, P, d, P, P, None, None, 0, P, d, P, d, None, None, 0, None),
        "rms_norm_backward": lambda ctx: L.rtb_rms_norm_backward(
            ctx, 2, d, P, d, P, None, P, d, None, 0, P, d, None, 0, None),
        "rms_norm_backward ": lambda ctx: L.rtb_rms_norm_backward_fp8(
            ctx, 2, d, P, d, P, blocks, P, None, P, d, None, 0, P, d, None, 0, None),
    }
    for name, call in calls.items():
        ctx = ctypes.create_string_buffer(4096)
        assert call(ctx) not in (rb._lib.RTB_OK, rb._lib.RTB_E_INVALID)
        assert rb._lib.last_error().startswith(name.strip()), rb._lib.last_error()


Q, R = ctypes.c_void_p(1 << 24), ctypes.c_void_p(1 << 26)


def forward(L, ctx, rows, x=P, ldx=64, residual=None, ldr=0, total=None, ldsum=0, y=Q, ldy=64):
    return L.rtb_rms_norm_fwd(ctx, rows, 64, x, ldx, residual, ldr, None, 1e-5, total, ldsum, y, ldy, None, None)


def backward(L, ctx, rows, dy=P, lddy=64, dsum=None, ldds=0, dx=Q, lddx=64):
    return L.rtb_rms_norm_backward(ctx, rows, 64, R, 64, R, None, dy, lddy, dsum, ldds, dx, lddx, None, 0, None)


IN_PLACE = [(forward, dict(y=P, ldy=65)), (forward, dict(y=P, ldx=80)), (forward, dict(residual=Q, ldr=96)),
            (forward, dict(residual=R, ldr=64, total=R, ldsum=72)), (forward, dict(total=P, ldsum=72)),
            (backward, dict(dx=P, lddx=65)), (backward, dict(dsum=Q, ldds=65))]


@pytest.mark.parametrize("call,args", IN_PLACE)
def test_in_place_rows_elsewhere_refused(rb, call, args):
    if torch.cuda.is_available():
        pytest.skip("checked where nothing can be launched")
    L = rb.lib()
    ctx = ctypes.create_string_buffer(4096)
    assert call(L, ctx, 2, **args) == rb._lib.RTB_E_INVALID
    assert "in place" in rb._lib.last_error()
    assert call(L, ctx, 1, **args) != rb._lib.RTB_E_INVALID  # one row lies where it lies
