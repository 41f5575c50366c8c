"""The root-mean-square norm where fp32 squares would not do: rows whose squares leave
fp32's range, and 8-bit values so near to the middle of two codes that the sum of squares
decides between them.

Tolerances, elementwise, U = 2^-24: squares and their sum are double, so that rstd has its
own rounding, U (2^-150 where it is no normal number); y = h hi w with hi rounded once and
two products, 3 U and what their product adds, and 2^-148 where y is no normal number."""
import pytest
import torch

from test_rms_gpu import EPS, U, check, reference

pytestmark = pytest.mark.gpu


def rounded8(y):
    """(values, scale bytes) of float64 rows: blocks of 128 columns by the smallest power of two
    that holds the largest magnitude within 448, each value rounded once, to nearest even."""
    rows, d = y.shape
    top = torch.nn.functional.pad(y.abs(), (0, -d % 128)).view(rows, -1, 128).amax(2)
    m, e = torch.frexp(top)  # 448 = 7/8 2^9
    e = torch.where(top > 0, (e - 9 + (m > 0.875).int()).clamp(min=-126), torch.zeros_like(e))
    v = torch.ldexp(y, -e.repeat_interleave(128, 1)[:, :d])
    step = torch.ldexp(torch.ones_like(v), torch.frexp(v).exponent.clamp(min=-5) - 4)
    return torch.round(v / step) * step, e + 127


def forward64(h, w, eps):
    h = h.double()
    rstd = (h.square().mean(1) + float(torch.tensor(eps, dtype=torch.float32))) ** -0.5
    y = h * rstd[:, None]
    return (y if w is None else y * w.double()), rstd


# a size for every number of threads and registers a row, with and without 16-byte rows
@pytest.mark.parametrize("rows,d", [(400, 64), (300, 77), (200, 256), (100, 300), (80, 512), (50, 1001), (40, 2048),
                                    (20, 4096), (20, 4097), (12, 8192), (8, 16384), (8, 16383), (6, 20001), (6, 20004)])
def test_fp8_next_to_the_middle_of_two_codes(gpu, rows, d):
    """Rows of any numbers, whose squares no fp32 sum holds exactly, and for each row a
    weight that puts its values within an fp32 rounding of the middle of two codes."""
    g = torch.Generator(device="cuda").manual_seed(61)
    for row in range(rows):
        h = torch.randn((1, d), device="cuda", generator=g)
        h = torch.where(h.abs() < 0.01, torch.ones_like(h), h) * float(torch.rand((), device="cuda", generator=g) + 0.1)
        _, rstd = forward64(h, None, EPS)
        k = torch.randint(-6, 8, (1, d), device="cuda", generator=g).double()
        middle = (1 + (2 * torch.randint(0, 6, (1, d), device="cuda", generator=g) + 1) / 16) * torch.pow(2.0, k)
        middle[:, ::128] = 232  # the block's largest
        w = (middle / (h.double() * rstd)).float()
        q, s, _, _ = gpu.rms_norm_fp8(h, w[0], EPS)
        want, byte = rounded8(forward64(h, w[0], EPS)[0])
        assert torch.equal(s.view(torch.uint8).int(), byte.int()) and torch.equal(q.double(), want)


@pytest.mark.parametrize("rows,d", [(1531, 1001), (32768, 512), (8192, 2048), (4096, 4096), (2048, 8192), (1024, 16384)])
def test_fp8_of_many_rows_rounded_once(gpu, rows, d):
    for seed in (1, 5):
        g = torch.Generator(device="cuda").manual_seed(seed)
        x = torch.randn((rows, d), device="cuda", generator=g) * (0.25 + 2 * torch.rand((rows, 1), device="cuda", generator=g))
        res = torch.randn((rows, d), device="cuda", generator=g)
        w = 1 + 0.1 * torch.randn(d, device="cuda", generator=g)
        q, s, h, _ = gpu.rms_norm_fp8(x, w, EPS, residual=res)
        want, byte = rounded8(forward64(h, w, EPS)[0])
        assert torch.equal(s.view(torch.uint8).int(), byte.int()) and torch.equal(q.double(), want)


@pytest.mark.parametrize("d", [1, 4, 64, 130, 300, 1001, 2048, 4096, 8192, 8193, 16383, 16384, 16385, 16388, 20001])
@pytest.mark.parametrize("size,eps", [(1e19, EPS), (1e20, EPS), (1e30, 1.0), (1e38, EPS), (3e38, 0.0), (1e-19, 0.0),
                                      (1e-23, 0.0), (1e-30, 0.0), (1e-37, 0.0), (1e-41, 0.0)])
def test_rows_of_any_magnitude(gpu, d, size, eps):
    g = torch.Generator(device="cuda").manual_seed(62)
    x = (torch.rand((5, d), device="cuda", generator=g) + 0.1).clamp(max=1.0) * size
    x *= 1 - 2 * torch.randint(0, 2, (5, d), device="cuda", generator=g)
    x[3, d // 2:] = 0.5  # beside values of another order
    w = 0.5 + torch.rand(d, device="cuda", generator=g)
    for weight in (w, None):
        y, h, rstd = gpu.rms_norm_fwd(x, weight, eps)
        q, s, _, r8 = gpu.rms_norm_fp8(x, weight, eps)
        wy, wr = forward64(x, weight, eps)
        assert torch.equal(h, x) and torch.equal(r8, rstd)
        big = wr >= 2.0 ** 128 * (1 - U / 2)  # (no number of fp32)
        assert bool((torch.isinf(rstd) == big).all())
        assert bool(((rstd.double() - wr).abs() <= U * wr * (1 + 2 * U) + 2.0 ** -150)[~big].all())
        assert bool(((y.double() - wy).abs() <= 3.01 * U * wy.abs() + 2.0 ** -148).all())
        small = wy.abs() < 2.0 ** -120  # (8 bits of these: half a unit of fp32's last place either way)
        want, byte = rounded8(wy)
        assert torch.equal(s.view(torch.uint8).int(), byte.int())
        assert torch.equal(torch.where(small, want, q.double()), want)


def test_gradients_of_large_rows(gpu):
    g = torch.Generator(device="cuda").manual_seed(63)
    for d in (300, 1024, 4096, 9000, 20000):
        x = torch.randn((7, d), device="cuda", generator=g) * 1e20
        dy, ds = (torch.randn((7, d), device="cuda", generator=g) for _ in range(2))
        w = 1 + 0.1 * torch.randn(d, device="cuda", generator=g)
        _, h, rstd = gpu.rms_norm_fwd(x, w, EPS)
        for grad_sum in (None, ds):
            want, bound = reference(x, rstd, w, dy, grad_sum)
            check(gpu.rms_norm_backward(h, rstd, dy, w, grad_sum), want, bound)
