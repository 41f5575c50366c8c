"""Operators of the 8-bit training block on tensors whose elements lie beyond 2^31
and bytes beyond 2^32: the first, some middle and the last rows against float64,
with the bounds of the small tests."""
import pytest
import torch

from test_fp8_gpu import operand, same_codes, ref_quantize, values64
from test_norm_backward_gpu import EPS, U, check, make, reference

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True)
def give_back():
    yield
    torch.cuda.empty_cache()


def repeated(t, rows):
    """t's rows over and over, `rows` of them."""
    out = torch.empty((rows, t.shape[1]), dtype=t.dtype, device="cuda")
    whole = rows // t.shape[0] * t.shape[0]
    out.view(torch.uint8 if t.element_size() == 1 else t.dtype)[:whole].view(
        -1, *t.shape).copy_(t.view(torch.uint8) if t.element_size() == 1 else t)
    if rows > whole:
        out.view(torch.uint8 if t.element_size() == 1 else t.dtype)[whole:] = (
            t.view(torch.uint8) if t.element_size() == 1 else t)[:rows - whole]
    return out


# rows of `d` floats that lie 2^31 elements and more apart, aligned and not
@pytest.mark.parametrize("rows,d", [(530000, 4096), (530000, 4099)])
def test_save_and_restore(gpu, rows, d):
    x0 = torch.randn((1000, d), generator=torch.Generator().manual_seed(1))
    x = repeated(x0.cuda(), rows)
    q, s = gpu.fp8_quantize(x)
    del x
    wq, ws = ref_quantize(x0, 1)
    last = rows // 1000 * 1000 - 1000
    for r in (0, 1000, last // 2000 * 1000, last):
        same_codes(q[r:r + 1000], wq)
        assert torch.equal(s[r:r + 1000].view(torch.uint8).cpu(), ws)
    y = gpu.fp8_dequantize(q, s)
    want = values64(wq, ws.view(torch.float8_e8m0fnu)).float().cuda()
    for r in (0, last // 2000 * 1000, last):
        assert torch.equal(y[r:r + 1000], want)


@pytest.mark.parametrize("d", [4096, 4099])
@pytest.mark.parametrize("saved", [False, True])
def test_norm_backward(gpu, d, saved):
    rows, n = 530000, 500
    x0, w, b, dy0 = make(n, d, 3)
    x, dy = repeated(x0, rows), repeated(dy0, rows)
    y, mean, rstd = gpu.layer_norm_fwd(x, w, b, EPS)
    y0, mean0, rstd0 = gpu.layer_norm_fwd(x0, w, b, EPS)
    for r in (0, rows // 2 // n * n, rows - n):
        assert torch.equal(y[r:r + n], y0) and torch.equal(mean[r:r + n], mean0)
    del y
    scale = None
    if saved:
        x, scale = gpu.fp8_quantize(x)
        x0 = gpu.fp8_dequantize(x[:n], scale[:n])
    dx, dw, db = gpu.layer_norm_backward(x, mean, rstd, dy, w, b, x_scale=scale)
    (wx, ww, wb), (ex, _, _) = reference(x0, mean0, rstd0, w, b, dy0, 0)
    for r in (0, rows // 2 // n * n, rows - n):
        assert bool(((dx[r:r + n].double() - wx).abs() <= ex).all())
    # the sums: rows / n times the block's, within the depth of a thread's chain
    dz, u = dy0.double(), (x0.double() - mean0.double()[:, None]) * rstd0.double()[:, None]
    steps = rows / 148 + 200
    for got, want, size in ((dw, ww, (dz * u).abs().sum(0)), (db, wb, dz.abs().sum(0))):
        assert bool(((got.double() - want * (rows / n)).abs() <= steps * U * size * (rows / n)).all())


# the output beyond 2^31 elements: rows along the tiles (stored by TMA, and
# directly), few rows against many columns; float scales
@pytest.mark.parametrize("m,n,k,floats", [(70001, 32768, 130, False), (70001, 32770, 130, False),
                                          (70001, 32770, 130, True), (65, 33100000, 128, False),
                                          (64, 33600000, 128, False), (9, 240000000, 16, False)])
def test_product(gpu, m, n, k, floats):
    a0, sa0 = operand(min(m, 1000), k, 1, 5)
    w0, sw0 = operand(1280, k, 1, 6)
    a, sa = repeated(a0, m), repeated(sa0, m)
    w, sw = repeated(w0, n), repeated(sw0, n)
    if floats:
        sw = torch.pow(2.0, sw.view(torch.uint8).float() - 127)
    c = gpu.fp8_matmul(a, sa, w.t(), sw.t())
    del w, sw
    A, W = values64(a0, sa0), values64(w0, sw0)
    z, S = A @ W.t(), A.abs() @ W.abs().t()
    bound = S * (8 * 2.0 ** -21 + 4 * 2.0 ** -24)  # 8 steps of 32 in two blocks
    for r in (0, m // 2 // 1000 * 1000, m // 1000 * 1000 - 1000):
        if r < 0:
            continue
        for t in (0, n // 2 // 1280 * 1280, n // 1280 * 1280 - 1280):
            got = c[r:r + 1000, t:t + 1280].double()
            assert bool(((got - z[:got.shape[0]]).abs() <= bound[:got.shape[0]]).all())
    if m < 1000:
        got = c[:, n - n % 1280:].double()
        assert bool(((got - z[:m, :n % 1280]).abs() <= bound[:m, :n % 1280]).all())
    else:
        got = c[m - m % 1000:, :1280].double()
        assert bool(((got - z[:m % 1000]).abs() <= bound[:m % 1000]).all())


def test_weight_gradient(gpu):
    m, n, k = 257, 33000, 66000
    a, sa = operand(m, k, 1, 7)
    grad = torch.randn((m, n), generator=torch.Generator().manual_seed(8)).cuda()
    db = gpu.matmul_backward_fp8(a, sa, None, grad, need_a=False)[1]
    A = values64(a, sa)
    for r in (0, 33000, k - 600):
        At = A[:, r:r + 600].t()
        z, S = At @ grad.double(), At.abs() @ grad.double().abs()
        assert bool(((db[r:r + 600].double() - z).abs() <= S * (24 * 2.0 ** -21 + 5 * 2.0 ** -24)).all())
