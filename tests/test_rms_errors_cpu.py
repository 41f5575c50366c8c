"""A backward pass that cannot be launched says which one it is (no GPU here: every launch
fails, on the host)."""
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
