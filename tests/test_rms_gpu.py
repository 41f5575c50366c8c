"""The root-mean-square norm (with the residual's addition, with an output in 8 bits,
and its backward pass) on the B200 against float64 restatements.

Tolerances, elementwise, U = 2^-24.  Forward: the sum is one rounding, so it is
compared for equality; the squares are added in at most 64 fp32 steps a thread, all of
one sign, and exactly enough from there on, so that rstd is off by half of that and
its own rounding: 34 U relative; y takes two more products.  Backward: dx adds the
product h = dy w, u times the mean of h u, and the residual stream's gradient; the
mean carries the rounding of a sum of d terms in at most d / 128 + 16 sequential
steps; u is off by U; dweight is a sum over the rows in at most `rows` steps."""
import pytest
import torch

from test_fp8_gpu import operand, same_codes, values64
from test_norm_backward_gpu import _two_threads

pytestmark = pytest.mark.gpu

EPS = 1e-5
U = 2.0 ** -24
E4M3, E8M0 = torch.float8_e4m3fn, torch.float8_e8m0fnu

# widths on both sides of every kernel's limit, with and without 16-byte rows
SHAPES = [(1, 1), (2, 3), (1, 32), (5, 100), (3, 128), (9, 129), (33, 256), (20, 257), (300, 512), (37, 513),
          (1000, 768), (16, 1024), (7, 1028), (5, 1001), (9, 1500), (64, 2048), (3, 2052), (130, 4096), (2, 4100),
          (7, 4097), (11, 6000), (6, 8192), (3, 8193), (5, 8200), (4, 16384), (3, 16383), (3, 16388), (2, 40001),
          (4000, 33), (2500, 256), (9, 4), (1, 16384)]


def make(rows, d, seed):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn((rows, d), generator=g) * (0.2 + 2 * torch.rand((rows, 1), generator=g)) + 0.3
    res = 2 * torch.randn((rows, d), generator=g)
    w = 1 + 0.3 * torch.randn(d, generator=g)
    return x.cuda(), res.cuda(), w.cuda()


def forward64(h, w):
    """(y, rstd) of the rounded sum h."""
    h = h.double()
    rstd = (h.square().mean(1) + EPS) ** -0.5
    y = h * rstd[:, None]
    return (y if w is None else y * w.double()), rstd


def check_forward(gpu, x, res, w):
    y, h, rstd = gpu.rms_norm_fwd(x, w, EPS, residual=res)
    want_h = x if res is None else x + res
    assert torch.equal(h, want_h)
    wy, wr = forward64(want_h, w)
    assert rstd.shape == x.shape[:-1] and bool(((rstd.double() - wr).abs() <= 34 * U * wr).all())
    assert bool(((y.double() - wy).abs() <= 36.5 * U * wy.abs() + 1e-44).all())
    return y, h, rstd


@pytest.mark.parametrize("rows,d", SHAPES)
@pytest.mark.parametrize("with_res", [False, True])
def test_forward(gpu, rows, d, with_res):
    x, res, w = make(rows, d, 1)
    check_forward(gpu, x, res if with_res else None, w)
    check_forward(gpu, x, res if with_res else None, None)


@pytest.mark.parametrize("rows,d", SHAPES)
@pytest.mark.parametrize("with_res", [False, True])
def test_forward_fp8(gpu, rows, d, with_res):
    """The 8-bit output is the float64 one rounded once: off by half of a code's step at
    most, and by what rstd is (34 U); the scale is the smallest power of two that holds
    the block within 448."""
    x, res, w = make(rows, d, 2)
    res = res if with_res else None
    y, h, rstd = gpu.rms_norm_fwd(x, w, EPS, residual=res)
    q, s, h8, r8 = gpu.rms_norm_fp8(x, w, EPS, residual=res)
    assert q.dtype == E4M3 and s.dtype == E8M0 and tuple(s.shape) == (rows, -(-d // 128))
    assert torch.equal(h8, h) and torch.equal(r8, rstd)
    check_codes(q, s, forward64(h, w)[0], 36 * U)


def check_codes(q, s, y, off):
    d = y.shape[1]
    wide = torch.nn.functional.pad(y.abs(), (0, -d % 128)).view(y.shape[0], -1, 128).amax(2)
    scale = torch.pow(2.0, s.view(torch.uint8).double() - 127)
    assert bool((wide <= 448 * scale * (1 + off)).all())
    assert bool(((wide > 224 * scale * (1 - off)) | (wide == 0) & (scale == 1)).all())
    scale = scale.repeat_interleave(128, 1)[:, :d]
    v = y / scale
    step = torch.pow(2.0, torch.floor(torch.log2(v.abs().clamp(min=2.0 ** -6))) - 3)
    assert bool(((q.double() - v).abs() <= step / 2 + off * v.abs()).all())


@pytest.mark.parametrize("rows,d", [(60, 64), (40, 77), (30, 128), (50, 300), (20, 1001), (10, 2048), (9, 4097), (5, 8192),
                                    (3, 16384), (2, 20001), (2, 20004)])
def test_forward_fp8_between_two_codes(gpu, rows, d):
    """Values within an fp32 rounding of the middle of two codes, where the nearer one
    shows only behind fp32's last place: whole numbers, so that the sum of squares is
    exact, and weights that put each value there."""
    g = torch.Generator().manual_seed(41)
    for row in range(rows):
        h = torch.randint(1, 100, (1, d), generator=g).double() * (2 * torch.randint(0, 2, (1, d), generator=g) - 1)
        rstd = (h.square().sum() / d + float(torch.tensor(EPS))) ** -0.5
        k = torch.randint(-6, 8, (1, d), generator=g).double()
        middle = (1 + (2 * torch.randint(0, 6, (1, d), generator=g) + 1) / 16) * torch.pow(2.0, k)
        middle[:, ::128] = 232  # the block's largest: its scale is 1
        w = (middle / (h * rstd)).float()
        y = h * rstd * w.double()
        q, s, _, _ = gpu.rms_norm_fp8(h.float().cuda(), w[0].cuda(), EPS)
        assert bool((s.view(torch.uint8) == 127).all())
        step = torch.pow(2.0, k - 3)
        step[:, ::128] = 16
        up, down = middle + step / 2, middle - step / 2
        assert bool((y != middle).all())
        assert torch.equal(q.double().cpu(), torch.where(y.abs() > middle, up, down) * torch.sign(y))


def reference(x, rstd, w, dy, ds):
    """(dx, dw) and their bounds, in float64."""
    x, dy, rstd = x.double(), dy.double(), rstd.double()[:, None]
    w = torch.ones(x.shape[1], device=x.device).double() if w is None else w.double()
    ds = torch.zeros_like(x) if ds is None else ds.double()
    u, h = x * rstd, dy * w
    m = (h * u).mean(1, keepdim=True)
    dx = rstd * (h - u * m) + ds
    steps = x.shape[1] / 128 + 16
    hu = (h * u).abs()
    e2 = (steps + 3) * hu.mean(1, keepdim=True)  # h, u and their product, and the sum
    dxe = rstd * (3 * h.abs() + u.abs() * e2 + 5 * (u * m).abs()) + 2 * (rstd * (h - u * m)).abs() + ds.abs()
    rows = x.shape[0]
    dwe = (rows + 8) * (dy * u).abs().sum(0)
    return (dx, (dy * u).sum(0)), (dxe * U, dwe * U)


def check(got, want, bound):
    for g, r, e, name in zip(got, want, bound, ("dx", "dw")):
        off = (g.double().reshape(r.shape) - r).abs()
        assert bool((off <= e + 1e-37).all()), (name, float((off / e.clamp(min=1e-37)).max()))


@pytest.mark.parametrize("rows,d", SHAPES)
@pytest.mark.parametrize("with_sum", [False, True])
@pytest.mark.parametrize("saved", [False, True])
def test_backward(gpu, rows, d, with_sum, saved):
    x, dy, w = make(rows, d, 3)
    ds = make(rows, d, 4)[0] if with_sum else None
    rstd = gpu.rms_norm_fwd(x, w, EPS)[2]
    scale = None
    source = x
    if saved:
        source, scale = gpu.fp8_quantize(x)
        x = gpu.fp8_dequantize(source, scale)
    for weight in (w, None):
        want, bound = reference(x, rstd, weight, dy, ds)
        check(gpu.rms_norm_backward(source, rstd, dy, weight, ds, x_scale=scale), want, bound)


def test_gradients_against_differences(gpu):
    """Central differences of the float64 forward (the norm's output and the sum, as
    the next layers read both), along random directions."""
    x, res, w = make(6, 40, 5)
    g = torch.Generator().manual_seed(6)
    dy, ds = torch.randn((6, 40), generator=g).cuda(), torch.randn((6, 40), generator=g).cuda()
    _, h, rstd = gpu.rms_norm_fwd(x, w, EPS, residual=res)
    dx, dw = gpu.rms_norm_backward(h, rstd, dy, w, ds)

    def loss(x, res, w):
        h = x + res
        return ((h * (h.square().mean(1, keepdim=True) + EPS) ** -0.5 * w) * dy.double()).sum() + (h * ds.double()).sum()

    args = [x.double(), res.double(), w.double()]
    for i, grad in enumerate((dx, dx, dw)):
        way = torch.randn(args[i].shape, generator=g).cuda().double()
        lo, hi = list(args), list(args)
        hi[i], lo[i] = args[i] + 1e-5 * way, args[i] - 1e-5 * way
        diff = (loss(*hi) - loss(*lo)) / 2e-5
        # differences: 1e-10 of the third derivatives; gradients: fp32
        assert abs(float((grad.double() * way).sum() - diff)) <= 1e-4 * float((grad.double() * way).abs().sum())


@pytest.mark.parametrize("d", [64, 333, 1024, 5000, 9000, 9001, 20000, 20001])
def test_in_place(gpu, d):
    """Outputs where inputs lie: the residual stream, the normed input, both; the
    gradient over either incoming one."""
    x, res, w = make(23, d, 7)
    y, h, rstd = gpu.rms_norm_fwd(x, w, EPS, residual=res)
    for out, total in ((None, "res"), ("x", None), ("x", "res"), ("res", "x"), (None, "x")):
        a = {"x": x.clone(), "res": res.clone(), None: None}
        gy, gh, gr = gpu.rms_norm_fwd(a["x"], w, EPS, residual=a["res"], out=a[out], out_sum=a[total])
        assert torch.equal(gy, y) and torch.equal(gh, h) and torch.equal(gr, rstd)
        assert (out is None or gy.data_ptr() == a[out].data_ptr()) and (total is None or gh.data_ptr() == a[total].data_ptr())
    r2 = res.clone()
    q, s, gh, gr = gpu.rms_norm_fp8(x, w, EPS, residual=r2, out_sum=r2)
    assert torch.equal(r2, h) and torch.equal(gr, rstd)
    same_codes(q, gpu.fp8_quantize(y)[0])
    z = x.clone()  # without a residual
    y0, same, r0 = gpu.rms_norm_fwd(x, w, EPS)
    assert same.data_ptr() == x.data_ptr()
    gpu.rms_norm_fwd(z, w, EPS, out=z)
    assert torch.equal(z, y0)
    copy = torch.empty_like(x)
    gpu.rms_norm_fwd(x, w, EPS, out_sum=copy)
    assert torch.equal(copy, x)
    dy, ds = make(23, d, 8)[:2]
    dx, dw = gpu.rms_norm_backward(h, rstd, dy, w, ds)
    for k in (0, 1):
        a = [dy.clone(), ds.clone()]
        gx, gw = gpu.rms_norm_backward(h, rstd, a[0], w, a[1], out_x=a[k])
        assert gx.data_ptr() == a[k].data_ptr() and torch.equal(gx, dx) and torch.equal(gw, dw)


def test_accumulate_and_parts(gpu):
    for d in (256, 333, 5000, 9000, 20000):
        x, dy, w = make(70, d, 9)
        ds = make(70, d, 10)[0]
        rstd = gpu.rms_norm_fwd(x, w, EPS)[2]
        full = gpu.rms_norm_backward(x, rstd, dy, w, ds)
        dx, dw = gpu.rms_norm_backward(x, rstd, dy, w, ds, need_x=False)
        assert dx is None and torch.equal(dw, full[1])
        dx, dw = gpu.rms_norm_backward(x, rstd, dy, w, ds, need_weight=False)
        assert dw is None and torch.equal(dx, full[0])
        g = torch.Generator().manual_seed(11)
        start = [torch.randn(t.shape, generator=g).cuda() for t in full]
        outs = [t.clone() for t in start]
        gpu.rms_norm_backward(x, rstd, dy, w, ds, out_x=outs[0], out_weight=outs[1], accumulate=True)
        for o, s, f in zip(outs, start, full):
            assert bool(((o - (s + f)).abs() <= 4 * U * (s.abs() + f.abs())).all())


def moved(t, offset, pad):
    """t with a row stride of d + pad, from element `offset` of its storage; NaN around."""
    rows, d = t.shape
    wide = torch.full((offset + rows * (d + pad),), float("nan"), device="cuda").to(t.dtype)
    view = wide.as_strided((rows, d), (d + pad, 1), offset)
    view.copy_(t)
    return view


@pytest.mark.parametrize("rows,d,offset,pad", [(950, 301, 1, 0), (130, 1000, 7, 3), (70, 4097, 0, 0), (46, 6001, 3, 5),
                                               (1, 129, 3, 1), (4000, 77, 13, 1), (2, 8191, 9, 2), (8, 1024, 4, 8),
                                               (3, 17000, 1, 0), (8, 1024, 0, 2)])
def test_rows_at_any_place(gpu, rows, d, offset, pad):
    """Row strides and bases off the 16-byte boundaries, each tensor's its own, and what
    lies around the outputs' rows stays as it was."""
    x, res, w = make(rows, d, 12)
    dy, ds = make(rows, d, 13)[:2]
    want = gpu.rms_norm_fwd(x, w, EPS, residual=res)
    y, h = moved(x, 0, pad), moved(x, offset, 0)
    got = gpu.rms_norm_fwd(moved(x, offset, pad), moved(w[None], offset, 0)[0], EPS, residual=moved(res, 0, pad), out=y, out_sum=h)
    for a, b, c in zip(got, want, (36.5 * 2, 0, 34 * 2)):  # (another order of the sum)
        assert bool(((a - b).abs() <= c * U * b.abs()).all())
    check_forward(gpu, moved(x, offset, pad), moved(res, offset, pad), w)
    base = y._base
    around = torch.ones_like(base, dtype=torch.bool)
    around.as_strided((rows, d), (d + pad, 1), 0)[:] = False
    assert bool(torch.isnan(base[around]).all())
    q, s, _, _ = gpu.rms_norm_fp8(moved(x, offset, pad), w, EPS, residual=res)
    ref = forward64(x + res, w)[0]
    step = torch.pow(2.0, s.view(torch.uint8).double() - 127).repeat_interleave(128, 1)[:, :d] * 2.0 ** -10
    assert bool(((values64(q, s) - ref).abs() <= torch.maximum(ref.abs() * 2.0 ** -4, step) + 40 * U * ref.abs()).all())
    want, bound = reference(x, want[2], w, dy, ds)
    rstd = gpu.rms_norm_fwd(x, w, EPS, residual=res)[2]
    check(gpu.rms_norm_backward(moved(x, offset, pad), rstd, moved(dy, offset, 0), w, moved(ds, 0, pad)), want, bound)
    xq, xs = gpu.fp8_quantize(x)
    want, bound = reference(gpu.fp8_dequantize(xq, xs), rstd, w, dy, ds)
    check(gpu.rms_norm_backward(moved(xq, offset, pad), rstd, dy, w, moved(ds, offset, pad), x_scale=xs), want, bound)


def test_shapes_and_expanded(gpu):
    x, res, w = make(24, 600, 14)
    x3 = x.view(4, 6, 600)
    y, h, rstd = gpu.rms_norm_fwd(x3, w, EPS, residual=res.view(4, 6, 600))
    flat = gpu.rms_norm_fwd(x, w, EPS, residual=res)
    assert y.shape == h.shape == x3.shape and rstd.shape == (4, 6) and torch.equal(y.view(24, 600), flat[0])
    q, s, _, _ = gpu.rms_norm_fp8(x3, w, EPS)
    assert q.shape == (4, 6, 600) and s.shape == (4, 6, 5)
    dx, dw = gpu.rms_norm_backward(h, rstd, x3, w, y)
    assert dx.shape == x3.shape and dw.shape == (600,)
    one = gpu.rms_norm_fwd(x[0], w, EPS)  # a single row
    assert one[0].shape == (600,) and one[2].shape == () and torch.equal(one[0], gpu.rms_norm_fwd(x, w, EPS)[0][0])
    row = x[:1].expand(24, 600)  # rows that share their memory
    y, h, rstd = gpu.rms_norm_fwd(row, w, EPS, residual=row)
    assert torch.equal(y, gpu.rms_norm_fwd(row.contiguous(), w, EPS, residual=row.contiguous())[0])
    t = make(30, 30, 15)[0].t()  # columns
    assert torch.equal(gpu.rms_norm_fwd(t)[0], gpu.rms_norm_fwd(t.contiguous())[0])
    grad = torch.ones((), device="cuda").expand(24, 600)
    want, bound = reference(x, flat[2], w, grad, grad)
    check(gpu.rms_norm_backward(x, flat[2], grad, w, grad), want, bound)


def test_empty_and_special_rows(gpu):
    w = torch.ones(40, device="cuda")
    e = torch.empty((0, 40), device="cuda")
    y, h, rstd = gpu.rms_norm_fwd(e, w, EPS, residual=e)
    q, s, _, _ = gpu.rms_norm_fp8(e, w, EPS)
    dx, dw = gpu.rms_norm_backward(e, rstd, e, w, e)
    assert y.shape == h.shape == q.shape == dx.shape == (0, 40) and s.shape == (0, 1) and bool((dw == 0).all())
    keep = torch.ones(40, device="cuda")
    gpu.rms_norm_backward(e, rstd, e, w, out_x=e, out_weight=keep, accumulate=True)
    assert bool((keep == 1).all())
    # a row of zeros, a NaN, an infinity: each in its own row
    x = torch.randn((5, 300), generator=torch.Generator().manual_seed(16)).cuda()
    x[1] = 0
    x[2, 7] = float("nan")
    x[3, 299] = float("inf")
    y, h, rstd = gpu.rms_norm_fwd(x, None, EPS)
    assert bool((y[1] == 0).all()) and abs(float(rstd[1]) - EPS ** -0.5) <= 2 * U * EPS ** -0.5
    assert bool(torch.isnan(y[2]).all()) and bool(torch.isnan(y[3, 299])) and bool((y[3, :299] == 0).all())
    assert bool(torch.isfinite(y[[0, 4]]).all())
    q, s, _, _ = gpu.rms_norm_fp8(x, None, EPS)
    wq, ws = gpu.fp8_quantize(y)
    same_codes(q, wq)
    assert torch.equal(s.view(torch.uint8), ws.view(torch.uint8)) and bool((s.view(torch.uint8)[1] == 127).all())
    dx, dw = gpu.rms_norm_backward(h, rstd, torch.ones_like(x))
    assert bool((dx[1] == rstd[1]).all()) and bool(torch.isnan(dx[2]).all()) and bool(torch.isfinite(dx[[0, 4]]).all())


# many rows for each group of threads, CTA and partial row, on every path
@pytest.mark.parametrize("rows,d", [(40000, 64), (40000, 77), (9500, 301), (9000, 256), (2600, 1000),
                                    (2600, 1001), (4099, 4096), (1999, 4097), (1500, 6000), (1500, 6001),
                                    (1203, 8192), (999, 9000), (999, 9001), (2411, 16500)])
@pytest.mark.parametrize("saved", [False, True])
def test_sums_over_rows_exactly(gpu, rows, d, saved):
    """With rstd 1 and small whole numbers every sum is a whole number below 2^24,
    exact in any order: a row that is lost, or added twice, shows."""
    g = torch.Generator(device="cuda").manual_seed(17)
    x = torch.randint(1, 5, (rows, d), device="cuda", generator=g).float()
    x *= 1 - 2 * torch.randint(0, 2, (rows, d), device="cuda", generator=g)
    dy = torch.randint(1, 4, (rows, d), device="cuda", generator=g).float()
    rstd = torch.ones(rows, device="cuda")
    dw = (dy.double() * x.double()).sum(0)
    scale = None
    if saved:
        x, scale = gpu.fp8_quantize(x)
    assert torch.equal(gpu.rms_norm_backward(x, rstd, dy, x_scale=scale, need_x=False)[1].double(), dw)
    start = torch.arange(d, device="cuda").float()
    gw = start.clone()
    gpu.rms_norm_backward(x, rstd, dy, x_scale=scale, out_x=torch.zeros_like(dy), out_weight=gw, accumulate=True)
    assert torch.equal(gw.double(), dw + start.double())


@pytest.mark.parametrize("d", [4096, 4099])
def test_beyond_2_31_elements(gpu, d):
    rows, n = 530000, 500
    x0, res0, w = make(n, d, 18)
    x = x0.repeat(rows // n, 1)
    y0, h0, r0 = gpu.rms_norm_fwd(x0, w, EPS, residual=res0)
    q0, s0 = gpu.fp8_quantize(y0)
    res = res0.repeat(rows // n, 1)
    y, h, rstd = gpu.rms_norm_fwd(x, w, EPS, residual=res, out=x, out_sum=res)
    for r in (0, rows // 2 // n * n, rows - n):
        assert torch.equal(y[r:r + n], y0) and torch.equal(h[r:r + n], h0) and torch.equal(rstd[r:r + n], r0)
    dx0 = gpu.rms_norm_backward(h0, r0, y0, w, h0)[0]
    dx, dw = gpu.rms_norm_backward(h, rstd, y, w, h, out_x=y)
    for r in (0, rows // 2 // n * n, rows - n):
        assert torch.equal(dx[r:r + n], dx0)
    u = h0.double() * r0.double()[:, None]
    want, size = (y0.double() * u).sum(0) * (rows / n), (y0.double() * u).abs().sum(0) * (rows / n)
    assert bool(((dw.double() - want).abs() <= (rows / 148 + 200) * U * size).all())
    del x, y, dx
    q, s, _, _ = gpu.rms_norm_fp8(h, w, EPS)
    q1, s1, _, _ = gpu.rms_norm_fp8(h0, w, EPS)
    for r in (0, rows - n):
        assert torch.equal(q[r:r + n].view(torch.uint8), q1.view(torch.uint8)) and torch.equal(s[r:r + n].view(torch.uint8), s1.view(torch.uint8))


def test_captured_and_side_stream(gpu):
    """Captured twice and replayed at the same time, with other inputs in the captured
    buffers; on a side stream; the same bits every time."""
    data = [make(700, 1024, 20 + i) for i in range(2)]

    def step(x, res, w):
        y, h, rstd = gpu.rms_norm_fwd(x, w, EPS, residual=res)
        q, s, _, _ = gpu.rms_norm_fp8(x, w, EPS, residual=res)
        return (y, h, rstd, q.view(torch.uint8), s.view(torch.uint8), *gpu.rms_norm_backward(h, rstd, x, w, res))

    want = [[t.clone() for t in step(*a)] for a in data]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = step(*data[0])
    side.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want[0]))
    graphs, outs, ins = [], [], []
    for i in range(2):
        ins.append([torch.zeros_like(t) for t in data[0]])
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(step(*ins[i]))
        graphs.append(g)
    for i in range(2):
        for a, b in zip(ins[i], data[i]):
            a.copy_(b)
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    for _ in range(3):
        for g, s in zip(graphs, streams):
            with torch.cuda.stream(s):
                g.replay()
    torch.cuda.synchronize()
    for i in range(2):
        assert all(torch.equal(a, b) for a, b in zip(outs[i], want[i]))


@pytest.mark.parametrize("widths", [(768, 4096), (2304, 1024), (1001, 4001), (9000, 16384)])
def test_two_threads(gpu, widths):
    def of(d):
        x, res, w = make(6, d, 30)
        _, h, rstd = gpu.rms_norm_fwd(x, w, EPS, residual=res)
        return lambda: (*gpu.rms_norm_fwd(x, w, EPS, residual=res), *gpu.rms_norm_backward(h, rstd, x, w, res))

    _two_threads(gpu, [of(d) for d in widths])


def test_feeds_the_8_bit_product(gpu):
    """Norm with an 8-bit output, product, and back: the weight gradient from the
    norm's output, the input's through the weight and the norm's checkpointed input.
    Each stage against float64 on what the stage before left."""
    x, res, nw = make(200, 640, 31)
    w, sw = operand(384, 640, 128, 32)
    grad = torch.randn((200, 384), generator=torch.Generator().manual_seed(33)).cuda()
    q, s, h, rstd = gpu.rms_norm_fp8(x, nw, EPS, residual=res)
    z = gpu.fp8_matmul(q, s, w.t(), sw.t())
    Y, W = values64(q, s), values64(w, sw)
    assert bool(((z.double() - Y @ W.t()).abs() <= Y.abs() @ W.abs().t() * 2.0 ** -18).all())
    y64 = forward64(h, nw)[0]
    assert float((Y - y64).norm() / y64.norm()) <= 2.0 ** -4
    dy, dw = gpu.matmul_backward_fp8(q, s, gpu.fp8_dequantize(w, sw).t().contiguous(), grad)
    assert float((dw.double() - Y.t() @ grad.double()).norm() / dw.double().norm()) <= 1e-6
    hq, hs = gpu.fp8_quantize(h)
    dx, dg = gpu.rms_norm_backward(hq, rstd, dy, nw, grad_sum=x, x_scale=hs)
    want, bound = reference(gpu.fp8_dequantize(hq, hs), rstd, nw, dy, x)
    check((dx, dg), want, bound)


def test_refusals(gpu):
    x, res, w = make(4, 128, 34)
    _, h, rstd = gpu.rms_norm_fwd(x, w)
    q, s = gpu.fp8_quantize(x)
    q128, s128 = gpu.fp8_quantize(x, 128)
    z = torch.zeros((), device="cuda")
    for call in (lambda: gpu.rms_norm_fwd(x, w[:5]), lambda: gpu.rms_norm_fp8(x, w[:5]),
                 lambda: gpu.rms_norm_fwd(z), lambda: gpu.rms_norm_fp8(z),
                 lambda: gpu.rms_norm_fwd(torch.zeros((4, 0), device="cuda")),
                 lambda: gpu.rms_norm_fwd(x.half()), lambda: gpu.rms_norm_fwd(x, residual=res[:3]),
                 lambda: gpu.rms_norm_fwd(x, residual=res.cpu()), lambda: gpu.rms_norm_fwd(x, residual=res.double()),
                 lambda: gpu.rms_norm_fwd(x, out=torch.zeros((4, 127), device="cuda")),
                 lambda: gpu.rms_norm_fwd(x, residual=res, out_sum=torch.zeros((128, 4), device="cuda").t()),
                 lambda: gpu.rms_norm_fwd(x, residual=res, out_sum=torch.zeros(128, device="cuda").expand(4, 128)),
                 lambda: gpu.rms_norm_backward(x, rstd, x[:, :5], w), lambda: gpu.rms_norm_backward(x, rstd[:3], x, w),
                 lambda: gpu.rms_norm_backward(x, rstd, x, w, res[:2]), lambda: gpu.rms_norm_backward(x, rstd, x, w[:3]),
                 lambda: gpu.rms_norm_backward(x, rstd, x, w, x_scale=s), lambda: gpu.rms_norm_backward(q, rstd, x, w),
                 lambda: gpu.rms_norm_backward(q128, rstd, x, w, x_scale=s128),
                 lambda: gpu.rms_norm_backward(q, rstd, x, w, x_scale=s.float()),
                 lambda: gpu.rms_norm_backward(x, rstd, x, w, accumulate=True),
                 lambda: gpu.rms_norm_backward(x, rstd, x, w, out_x=torch.zeros((4, 64), device="cuda"))):
        with pytest.raises(ValueError):
            call()
    both = torch.zeros_like(x)
    with pytest.raises(gpu.RtbError, match="one place"):
        gpu.rms_norm_fwd(x, w, residual=res, out=both, out_sum=both)


@pytest.mark.parametrize("d", [4, 100, 301, 512, 1001, 1024, 4096, 4097, 8192, 8191])
def test_backward_of_one_cta_and_more(gpu, d):
    """Row counts on both sides of what one CTA takes alone, with and without the
    reduced gradient, added to what is there."""
    for rows in (1, 2, 3, 4, 5, 8, 9, 16, 17, 32, 33):
        x, dy, w = make(rows, d, 51)
        rstd = forward64(x, None)[1].float()
        want, bound = reference(x, rstd, w, dy, x)
        got = gpu.rms_norm_backward(x, rstd, dy, w, grad_sum=x)
        check(got, want, bound)
        only = gpu.rms_norm_backward(x, rstd, dy, w, grad_sum=x, need_weight=False)
        assert only[1] is None and torch.equal(only[0], got[0])
        only = gpu.rms_norm_backward(x, rstd, dy, w, need_x=False)
        assert only[0] is None and torch.equal(only[1], got[1])
        out = torch.ones(d, device="cuda")
        gpu.rms_norm_backward(x, rstd, dy, w, need_x=False, out_weight=out, accumulate=True)
        assert torch.equal(out, 1 + got[1])
