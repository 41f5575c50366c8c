"""Layer norm's training forward and its backward pass on the B200 against
float64 restatements.

Tolerances, elementwise: an fp32 result is within c * 2^-24 of the magnitudes
that enter it.  dx adds three terms (h, its mean, u times the mean of h u), each
a product of up to three rounded factors: c = 16, and the two means carry the
rounding of a sum of d terms in at most d / 128 + 16 sequential steps (fewer in
every kernel).  The weight's and bias's gradients are sums over the rows in at
most `rows` sequential steps; u itself is off by 2^-23 (|x| + |mean|) rstd."""
import pytest
import torch

pytestmark = pytest.mark.gpu

EPS = 1e-5
U = 2.0 ** -24


def make(rows, d, seed, offset=0.5):
    g = torch.Generator().manual_seed(seed)
    x = (torch.randn((rows, d), generator=g) * (0.2 + 2 * torch.rand((rows, 1), generator=g)) + offset)
    w = 1 + 0.3 * torch.randn(d, generator=g)
    b = 0.3 * torch.randn(d, generator=g)
    dy = torch.randn((rows, d), generator=g)
    return x.cuda(), w.cuda(), b.cuda(), dy.cuda()


def activation64(z, act):
    return (z, torch.relu(z), torch.sigmoid(z), torch.tanh(z))[act]


def slope64(z, act):
    s = torch.sigmoid(z)
    return (torch.ones_like(z), (z > 0).double(), s * (1 - s), 1 - torch.tanh(z) ** 2)[act]


def reference(x, mean, rstd, w, b, dy, act):
    """(dx, dw, db) and the magnitudes that each is rounded at, in float64."""
    x, dy, mean, rstd = x.double(), dy.double(), mean.double()[:, None], rstd.double()[:, None]
    w = torch.ones(x.shape[1], device=x.device).double() if w is None else w.double()
    b = torch.zeros_like(w) if b is None else b.double()
    u = (x - mean) * rstd
    z = u * w + b
    dz = dy * slope64(z, act)
    h = dz * w
    m1, m2 = h.mean(1, keepdim=True), (h * u).mean(1, keepdim=True)
    dx = rstd * (h - m1 - u * m2)
    ue = 2 * (x.abs() + mean.abs()) * rstd + u.abs()  # u's error, in units of U
    # slopes of sigmoid and tanh move by at most the error of z, times a
    # second derivative below 1, and the functions' own few ulp
    ze = ue * w.abs() + 2 * z.abs() if act >= 2 else torch.zeros_like(z)
    he = (dy * w).abs() * (ze + 16 * (act >= 2)) + 4 * h.abs()
    steps = x.shape[1] / 128 + 16
    e1 = he.mean(1, keepdim=True) + steps * h.abs().mean(1, keepdim=True)
    hu = (h * u).abs()
    e2 = ((he * u.abs()) + h.abs() * ue).mean(1, keepdim=True) + steps * hu.mean(1, keepdim=True)
    dxe = rstd * (he + e1 + ue * m2.abs() + u.abs() * e2 + 4 * (h.abs() + m1.abs() + (u * m2).abs()))
    rows = x.shape[0]
    dwe = (he / w.abs().clamp(min=1e-30) * u.abs() + dz.abs() * ue).sum(0) + (rows + 8) * (dz * u).abs().sum(0)
    dbe = (he / w.abs().clamp(min=1e-30)).sum(0) + (rows + 8) * dz.abs().sum(0)
    return (dx, (dz * u).sum(0), dz.sum(0)), (dxe * U, dwe * U, dbe * U)


def check(got, want, bound):
    for g, r, e, name in zip(got, want, bound, ("dx", "dw", "db")):
        off = (g.double().reshape(r.shape) - r).abs()
        assert bool((off <= e + 1e-37).all()), (name, float((off / e.clamp(min=1e-37)).max()))


# widths on both sides of every kernel's limit, with and without 16-byte rows
SHAPES = [(1, 1), (2, 3), (1, 32), (5, 100), (3, 128), (9, 500), (300, 512), (37, 513), (1000, 768),
          (7, 1024), (5, 1001), (9, 1500), (64, 2048), (3, 2052), (130, 4096), (2, 4100), (11, 6000),
          (6, 8192), (3, 8193), (5, 8200), (4, 16384), (3, 16388), (2, 40000), (4000, 33), (2500, 256)]


@pytest.mark.parametrize("rows,d", SHAPES)
@pytest.mark.parametrize("act", [0, 3])
def test_forward_statistics(gpu, rows, d, act):
    x, w, b, _ = make(rows, d, 1)
    y, mean, rstd = gpu.layer_norm_fwd(x, w, b, EPS, act)
    assert torch.equal(y, gpu.layer_norm(x, w, b, EPS, act))  # the same pass
    x64 = x.double()
    m = x64.mean(1)
    v = ((x64 - m[:, None]) ** 2).mean(1)
    steps = d / 128 + 16
    assert bool(((mean.double() - m).abs() <= steps * U * x64.abs().mean(1)).all())
    r = (v + EPS) ** -0.5
    # the deviations are rounded at |x|: relative to the standard deviation
    e = 2 * steps * U + 4 * U * (x64.abs() + m.abs()[:, None]).amax(1) * r
    assert bool(((rstd.double() - r).abs() <= e * r).all())


@pytest.mark.parametrize("rows,d", SHAPES)
@pytest.mark.parametrize("act", [0, 3])
def test_backward(gpu, rows, d, act):
    x, w, b, dy = make(rows, d, 2)
    _, mean, rstd = gpu.layer_norm_fwd(x, w, b, EPS, act)
    want, bound = reference(x, mean, rstd, w, b, dy, act)
    check(gpu.layer_norm_backward(x, mean, rstd, dy, w, b, act), want, bound)


@pytest.mark.parametrize("rows,d", SHAPES)
def test_backward_from_checkpoint(gpu, rows, d):
    x, w, b, dy = make(rows, d, 3)
    _, mean, rstd = gpu.layer_norm_fwd(x, w, b, EPS)
    q, s = gpu.fp8_quantize(x)
    want, bound = reference(gpu.fp8_dequantize(q, s), mean, rstd, w, b, dy, 0)
    check(gpu.layer_norm_backward(q, mean, rstd, dy, w, b, x_scale=s), want, bound)


@pytest.mark.parametrize("act", [0, 1, 2, 3])
@pytest.mark.parametrize("affine", [False, True])
@pytest.mark.parametrize("d", [384, 1001])
@pytest.mark.parametrize("saved", [False, True])
def test_backward_activations(gpu, act, affine, d, saved):
    x, w, b, dy = make(50, d, 4)
    if not affine:
        w = b = None
    _, mean, rstd = gpu.layer_norm_fwd(x, w, b, EPS, act)
    s = None
    x64 = x
    if saved:
        x, s = gpu.fp8_quantize(x)
        x64 = gpu.fp8_dequantize(x, s)
    if act == 1:  # the derivative jumps at 0: keep z away from it by more than its error
        z = (x64 - mean[:, None]) * rstd[:, None] * (1 if w is None else w) + (0 if b is None else b)
        dy = torch.where(z.abs() < 1e-4, torch.zeros_like(dy), dy)
    want, bound = reference(x64, mean, rstd, w, b, dy, act)
    check(gpu.layer_norm_backward(x, mean, rstd, dy, w, b, act, x_scale=s), want, bound)


def test_gradients_against_differences(gpu):
    """Central differences of the float64 forward, along random directions."""
    x, w, b, dy = make(6, 40, 5)
    act = 3
    _, mean, rstd = gpu.layer_norm_fwd(x, w, b, EPS, act)
    dx, dw, db = gpu.layer_norm_backward(x, mean, rstd, dy, w, b, act)

    def loss(x, w, b):
        m = x.mean(1, keepdim=True)
        v = ((x - m) ** 2).mean(1, keepdim=True)
        return (torch.tanh((x - m) / torch.sqrt(v + EPS) * w + b) * dy.double()).sum()

    args = [x.double(), w.double(), b.double()]
    g = torch.Generator().manual_seed(6)
    for i, grad in enumerate((dx, dw, db)):
        way = torch.randn(args[i].shape, generator=g).cuda().double()
        lo, hi = list(args), list(args)
        hi[i], lo[i] = args[i] + 1e-5 * way, args[i] - 1e-5 * way
        diff = (loss(*hi) - loss(*lo)) / 2e-5
        # differences: 1e-10 of the third derivatives; gradients: fp32
        assert abs(float((grad.double() * way).sum() - diff)) <= 1e-4 * float((grad.double() * way).abs().sum())


def test_accumulate_and_parts(gpu):
    for d in (256, 333, 5000):
        x, w, b, dy = make(70, d, 7)
        _, mean, rstd = gpu.layer_norm_fwd(x, w, b, EPS)
        full = gpu.layer_norm_backward(x, mean, rstd, dy, w, b)
        # any subset of the outputs, the same bits
        dx, dw, db = gpu.layer_norm_backward(x, mean, rstd, dy, w, b, need_x=False)
        assert dx is None and torch.equal(dw, full[1]) and torch.equal(db, full[2])
        dx, dw, db = gpu.layer_norm_backward(x, mean, rstd, dy, w, b, need_weight=False)
        assert dw is None and torch.equal(dx, full[0]) and torch.equal(db, full[2])
        dx, dw, db = gpu.layer_norm_backward(x, mean, rstd, dy, w, b, need_weight=False,
                                             need_bias=False)
        assert torch.equal(dx, full[0])
        g = torch.Generator().manual_seed(8)
        start = [torch.randn(t.shape, generator=g).cuda() for t in full]
        outs = [t.clone() for t in start]
        gpu.layer_norm_backward(x, mean, rstd, dy, w, b, out_x=outs[0], out_weight=outs[1],
                                out_bias=outs[2], accumulate=True)
        for o, s, f in zip(outs, start, full):
            assert bool(((o - (s + f)).abs() <= 4 * U * (s.abs() + f.abs())).all())


def test_strides(gpu):
    """Rows of wider matrices, an unaligned base, an expanded gradient, more
    dimensions."""
    x, w, b, dy = make(24, 600, 9)
    for cols in (slice(0, 512), slice(1, 513), slice(3, 100)):
        xs, ds, ws, bs = x[:, cols], dy[:, cols], w[cols], b[cols]
        _, mean, rstd = gpu.layer_norm_fwd(xs, ws, bs, EPS)
        want, bound = reference(xs, mean, rstd, ws, bs, ds, 0)
        check(gpu.layer_norm_backward(xs, mean, rstd, ds, ws, bs), want, bound)
        one = torch.ones((), device="cuda").expand(xs.shape)
        want, bound = reference(xs, mean, rstd, ws, bs, one, 0)
        check(gpu.layer_norm_backward(xs, mean, rstd, one, ws, bs), want, bound)
    x3, d3 = x.view(4, 6, 600), dy.view(4, 6, 600)
    y, mean, rstd = gpu.layer_norm_fwd(x3, w, b, EPS)
    assert y.shape == x3.shape and mean.shape == (4, 6)
    dx, dw, db = gpu.layer_norm_backward(x3, mean, rstd, d3, w, b)
    flat = gpu.layer_norm_backward(x, mean.view(-1), rstd.view(-1), dy, w, b)
    assert dx.shape == x3.shape and torch.equal(dx.view(24, 600), flat[0])
    # in place: y over x
    z = x.clone()
    gpu.layer_norm_fwd(z, w, b, EPS, out=z)
    assert torch.equal(z, y.view(24, 600))


def test_empty_and_special_rows(gpu):
    w, b = torch.ones(40, device="cuda"), torch.zeros(40, device="cuda")
    e = torch.empty((0, 40), device="cuda")
    y, mean, rstd = gpu.layer_norm_fwd(e, w, b, EPS)
    dx, dw, db = gpu.layer_norm_backward(e, mean, rstd, e, w, b)
    assert y.shape == dx.shape == (0, 40)
    assert bool((dw == 0).all()) and bool((db == 0).all())
    keep = torch.ones(40, device="cuda")
    gpu.layer_norm_backward(e, mean, rstd, e, w, b, out_x=e, out_weight=keep,
                            out_bias=torch.ones(40, device="cuda"), accumulate=True)
    assert bool((keep == 1).all())
    # a constant row: u = 0, rstd = eps^-1/2
    x = torch.full((3, 40), 2.5, device="cuda")
    x[1, 4] = float("nan")
    dy = torch.randn((3, 40), generator=torch.Generator().manual_seed(1)).cuda()
    y, mean, rstd = gpu.layer_norm_fwd(x, w, b, EPS)
    dx, dw, db = gpu.layer_norm_backward(x, mean, rstd, dy, w, b)
    assert bool(torch.isnan(dx[1]).all()) and bool(torch.isfinite(dx[[0, 2]]).all())
    assert bool(torch.isnan(dw).all()) and bool(torch.isfinite(db).all())
    want = (dy[0] - dy[0].mean()) * EPS ** -0.5
    assert bool(((dx[0] - want).abs() <= 1e-5 * want.abs().max()).all())


def test_repeatable_and_captured(gpu):
    x, w, b, dy = make(700, 1024, 10)
    _, mean, rstd = gpu.layer_norm_fwd(x, w, b, EPS)
    first = gpu.layer_norm_backward(x, mean, rstd, dy, w, b)
    xi, di = torch.zeros_like(x), torch.zeros_like(dy)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out = gpu.layer_norm_backward(xi, mean, rstd, di, w, b)
    xi.copy_(x)
    di.copy_(dy)
    for _ in range(2):
        g.replay()
        again = gpu.layer_norm_backward(x, mean, rstd, dy, w, b)
        torch.cuda.synchronize()
        for a, o, f in zip(again, out, first):
            assert torch.equal(a, f) and torch.equal(o, f)


def test_refusals(gpu):
    x, w, b, dy = make(4, 128, 11)
    _, mean, rstd = gpu.layer_norm_fwd(x, w, b, EPS)
    q, s = gpu.fp8_quantize(x)
    q128, s128 = gpu.fp8_quantize(x, 128)
    for call in (lambda: gpu.layer_norm_fwd(x, w[:5], b),
                 lambda: gpu.layer_norm_fwd(torch.zeros((), device="cuda")),
                 lambda: gpu.layer_norm_fwd(x, out=torch.zeros((4, 127), device="cuda")),
                 lambda: gpu.layer_norm_backward(x, mean, rstd, dy[:, :5], w, b),
                 lambda: gpu.layer_norm_backward(x, mean[:3], rstd, dy, w, b),
                 lambda: gpu.layer_norm_backward(x, mean, rstd, dy, w, b[:3]),
                 lambda: gpu.layer_norm_backward(x, mean, rstd, dy, w, b, x_scale=s),
                 lambda: gpu.layer_norm_backward(q, mean, rstd, dy, w, b),
                 lambda: gpu.layer_norm_backward(q128, mean, rstd, dy, w, b, x_scale=s128),
                 lambda: gpu.layer_norm_backward(q, mean, rstd, dy, w, b, x_scale=s.float()),
                 lambda: gpu.layer_norm_backward(x, mean, rstd, dy, w, b, accumulate=True),
                 lambda: gpu.layer_norm_backward(x.half(), mean, rstd, dy, w, b)):
        with pytest.raises(ValueError):
            call()
    with pytest.raises(gpu.RtbError):
        gpu.layer_norm_backward(x, mean, rstd, dy, w, b, 5)


def test_layer_norm_of_an_expanded_row(gpu):
    """layer_norm of rows that share their memory (a stride of 0) reads them as
    they are."""
    row = torch.randn((1, 300), generator=torch.Generator().manual_seed(1)).cuda()
    y = gpu.layer_norm(row.expand(50, 300))
    assert torch.equal(y, gpu.layer_norm(row.expand(50, 300).contiguous()))


# rows that begin at any byte, several of them to each group of threads
@pytest.mark.parametrize("rows,d,offset,pad", [(9500, 301, 1, 0), (1300, 1000, 7, 3), (700, 4097, 0, 0),
                                               (460, 6001, 15, 5), (1, 129, 3, 1), (40000, 77, 13, 1),
                                               (2, 8191, 9, 2)])
@pytest.mark.parametrize("act", [0, 2])
@pytest.mark.parametrize("saved", [False, True])
def test_rows_at_any_byte(gpu, rows, d, offset, pad, act, saved):
    x, w, b, dy = make(rows, d, 11)
    _, mean, rstd = gpu.layer_norm_fwd(x, w, b, EPS, act)

    def moved(t):
        """t with a row stride of d + pad, from element `offset` of its storage;
        NaN around the rows."""
        wide = torch.full((offset + rows * (d + pad),), float("nan"), device="cuda").to(t.dtype)
        view = wide.as_strided((rows, d), (d + pad, 1), offset)
        view.copy_(t)
        return view

    scale = None
    if saved:
        q, scale = gpu.fp8_quantize(x)
        x, source = gpu.fp8_dequantize(q, scale), moved(q)
    else:
        source = moved(x)
    want, bound = reference(x, mean, rstd, w, b, dy, act)
    check(gpu.layer_norm_backward(source, mean, rstd, moved(dy), w, b, act, x_scale=scale), want, bound)


def test_a_row_of_more_than_2_30_columns(gpu):
    """One row whose two partial sums lie 2^30 floats and more apart: with mean 0
    and rstd 1, u = x, so that the sums are x * x and x, to the bit."""
    d = 2 ** 30 + 64
    x = torch.empty((1, d), device="cuda")
    x.view(-1, 64)[:] = torch.arange(1, 65, device="cuda").float()
    x[0, ::1009] = -3.25
    zero, one = torch.zeros(1, device="cuda"), torch.ones(1, device="cuda")
    _, dw, db = gpu.layer_norm_backward(x, zero, one, x, need_x=False)
    assert torch.equal(db, x[0])
    del db
    assert torch.equal(dw, (x * x)[0])


# widths of one kernel that need unlike amounts of shared memory
@pytest.mark.parametrize("widths", [(768, 4096), (2304, 1024), (1001, 4001)])
@pytest.mark.parametrize("saved", [False, True])
def test_two_threads_with_unlike_widths(gpu, widths, saved):
    _two_threads(gpu, [_backward_of(gpu, d, saved) for d in widths])


def test_two_threads_forward(gpu):
    # (rows off the 16-byte boundaries, staged in shared memory)
    def forward(d):
        x, w, b, _ = make(4, d, 13)
        return lambda: gpu.layer_norm_fwd(x, w, b, EPS)

    _two_threads(gpu, [forward(12301), forward(16383)])


def _backward_of(gpu, d, saved):
    x, w, b, dy = make(6, d, 12)
    _, mean, rstd = gpu.layer_norm_fwd(x, w, b, EPS)
    scale = None
    if saved:
        x, scale = gpu.fp8_quantize(x)
    return lambda: gpu.layer_norm_backward(x, mean, rstd, dy, w, b, x_scale=scale)


def _two_threads(gpu, calls):
    """Both calls over and over, each in a thread and on a stream of its own."""
    import threading
    want = [call() for call in calls]
    torch.cuda.synchronize()
    got, errors = [None, None], []
    streams = [torch.cuda.Stream() for _ in calls]
    start = threading.Barrier(len(calls))

    def work(i):
        try:
            start.wait()
            with torch.cuda.stream(streams[i]):
                for _ in range(1500):
                    got[i] = calls[i]()
        except Exception as e:
            errors.append(e)

    threads = [threading.Thread(target=work, args=(i,)) for i in range(len(calls))]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    torch.cuda.synchronize()
    assert not errors, errors
    for a, b in zip(got, want):
        assert all(torch.equal(x, y) for x, y in zip(a, b))


@pytest.mark.parametrize("d", [100, 1000, 1001, 5000, 5001, 9000, 9001, 20000])
@pytest.mark.parametrize("act", [2, 3])
@pytest.mark.parametrize("saved", [False, True])
def test_slopes_of_saturated_activations(gpu, d, act, saved):
    """One row with u = 0, so that z is the bias and dbias = dy act'(z): the slope
    keeps its relative accuracy where the activation is next to its limits.  In
    units of 2^-24, for e / (1 + e (2 + e)): the exponential 4 (2 ulp; the slope moves
    by at most as much), the denominator 1.75 (2 + e rounded, times at most 3/4, and
    the sum), its reciprocal 2 (1 ulp), the two products with e and dy 2; z stays
    where e is a normal number."""
    most = 80.0 if act == 2 else 40.0
    g = torch.Generator().manual_seed(15)
    z = most * (2 * torch.rand(d, generator=g) - 1)
    z[:6] = torch.tensor([0.0, -0.0, most, -most, 1e-6, 12.0])
    dy = (0.5 + torch.rand((1, d), generator=g)).cuda()
    x, z, one = torch.zeros((1, d), device="cuda"), z.cuda(), torch.ones(1, device="cuda")
    scale = None
    if saved:
        x, scale = gpu.fp8_quantize(x)
    db = gpu.layer_norm_backward(x, torch.zeros_like(one), one, dy, None, z, act, x_scale=scale)[2]
    z = z.double()
    slope = torch.sigmoid(z) * torch.sigmoid(-z) if act == 2 else torch.cosh(z) ** -2
    want = dy[0].double() * slope
    assert bool(((db.double() - want).abs() <= 9.75 * U * want).all())
    # and at the ends of the range, where the slope is 0
    ends = torch.tensor([3e38, -3e38, float("inf"), -float("inf")] * 25, device="cuda")
    x = torch.zeros((1, 100), device="cuda")
    db = gpu.layer_norm_backward(x, torch.zeros_like(one), one, torch.ones_like(x), None, ends, act)[2]
    assert bool((db == 0).all())


# many rows for each group of threads, CTA and partial row, on every path
@pytest.mark.parametrize("rows,d", [(40000, 64), (40000, 77), (9500, 301), (9000, 256), (2600, 1000),
                                    (2600, 1001), (4099, 4096), (1999, 4097), (1500, 6000), (1500, 6001),
                                    (1203, 8192), (999, 9000), (999, 9001), (2411, 16500)])
@pytest.mark.parametrize("saved", [False, True])
def test_sums_over_rows_exactly(gpu, rows, d, saved):
    """With mean 0, rstd 1 and small whole numbers every sum is a whole number
    below 2^24, exact in any order: a row that is lost, or added twice, shows."""
    g = torch.Generator(device="cuda").manual_seed(16)
    x = torch.randint(1, 5, (rows, d), device="cuda", generator=g).float()
    x *= 1 - 2 * torch.randint(0, 2, (rows, d), device="cuda", generator=g)
    dy = torch.randint(1, 4, (rows, d), device="cuda", generator=g).float()
    mean, rstd = torch.zeros(rows, device="cuda"), torch.ones(rows, device="cuda")
    dw, db = (dy.double() * x.double()).sum(0), dy.double().sum(0)
    scale = None
    if saved:
        x, scale = gpu.fp8_quantize(x)
    _, gw, gb = gpu.layer_norm_backward(x, mean, rstd, dy, x_scale=scale, need_x=False)
    assert torch.equal(gw.double(), dw) and torch.equal(gb.double(), db)
    start = torch.arange(d, device="cuda").float()
    gw, gb = start.clone(), -start
    gpu.layer_norm_backward(x, mean, rstd, dy, x_scale=scale, out_x=torch.zeros_like(dy), out_weight=gw,
                            out_bias=gb, accumulate=True)
    assert torch.equal(gw.double(), dw + start.double()) and torch.equal(gb.double(), db - start.double())
