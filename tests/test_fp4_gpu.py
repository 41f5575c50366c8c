"""4-bit block-scaled tensors on the B200: writing and restoring them and their
product, against plain restatements in float64.

Saving is exact arithmetic with one rounding, so its bytes are compared for equality.
Products are held elementwise to gamma * S, S = sum of |a||b| over the contraction:
products of codes are exact (and with the scales too, as long as they stay in fp32's
range); the tensor core adds steps of 64, each within 2^-24 of the running sum, on
average half of the unit's S, at most 64 of them (2^-19 together) before their sum is
added in fp32, which happens after every 2048 elements at least: (K / 2048 + 2)
2^-24."""
import numpy as np
import pytest
import torch

from test_norm_backward_gpu import _two_threads

pytestmark = pytest.mark.gpu

E2M1, E8M0 = torch.float4_e2m1fn_x2, torch.float8_e8m0fnu
GRID = np.array([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0])
INF, NAN = float("inf"), float("nan")


def ref_quantize(x):
    """(bytes of two codes, scale bytes) of a matrix by the format's definition, on the CPU."""
    x = x.cpu().double().numpy()
    rows, cols = x.shape
    cb = -(-cols // 32)
    full = np.zeros((rows, cb * 32))
    full[:, :cols] = x
    blocks = full.reshape(rows, cb, 32)
    bad = ~np.isfinite(blocks).all(axis=2)
    clean = np.where(bad[:, :, None], 0.0, blocks)
    top = np.abs(clean).max(axis=2)
    m, e = np.frexp(top)  # top = m 2^e, m in [1/2, 1); 6 = 3/4 2^3
    exponent = np.where(top > 0, np.maximum(np.where(m <= 0.75, e - 3, e - 2), -126), 0)
    v = clean * np.exp2(-exponent.astype(np.float64))[:, :, None]
    a = np.abs(v)
    # the nearest value of the grid; halfway: the even code
    hi = np.searchsorted(GRID, a).clip(0, 7)
    lo = (hi - 1).clip(0, 7)
    dl, dh = a - GRID[lo], GRID[hi] - a
    code = np.where((dl < dh) | ((dl == dh) & (lo % 2 == 0)), lo, hi)
    code = np.where(GRID[hi] == a, hi, code) + 8 * np.signbit(v)
    code[bad] = 0
    code = code.reshape(rows, cb * 32).astype(np.uint8)
    byte = np.where(bad, 255, exponent + 127).astype(np.uint8)
    q = (code[:, 0::2] | (code[:, 1::2] << 4))[:, :(cols + 1) // 2]
    return torch.from_numpy(np.ascontiguousarray(q)), torch.from_numpy(byte)


def values64(q, scale, cols=None):
    """The float64 values of (q, scale)."""
    byte = q.view(torch.uint8).long()
    code = torch.stack((byte & 15, byte >> 4), 2).view(byte.shape[0], -1)
    v = torch.from_numpy(GRID).to(q.device)[code & 7] * (1 - 2 * (code >> 3))
    sb = scale.view(torch.uint8).double()
    s = torch.where(sb == 255, torch.full_like(sb, NAN), torch.pow(2.0, sb - 127))
    return (v * s.repeat_interleave(32, 1)[:, :v.shape[1]])[:, :cols]


def spread(shape, seed, low=-6.0, high=6.0):
    """Normal values with magnitudes spread over a few powers of ten."""
    g = torch.Generator().manual_seed(seed)
    return torch.randn(shape, generator=g) * torch.pow(10.0, low + (high - low) * torch.rand((shape[0], 1), generator=g))


def operand(rows, k, seed):
    """Any codes, with scales of a few powers of two apart."""
    g = torch.Generator(device="cuda").manual_seed(seed)
    q = torch.randint(0, 256, (rows, k // 2), device="cuda", generator=g, dtype=torch.uint8).view(E2M1)
    s = torch.randint(122, 132, (rows, -(-k // 32)), device="cuda", generator=g, dtype=torch.uint8).view(E8M0)
    return q, s


def same(got, want):
    q, s = got
    return torch.equal(q.view(torch.uint8).cpu(), want[0]) and torch.equal(s.view(torch.uint8).cpu(), want[1])


# ------------------------------------------------------------------ save and restore

SHAPES = [(1, 1), (1, 2), (1, 32), (3, 33), (7, 1000), (130, 64), (128, 128), (257, 385), (64, 4096), (5, 31),
          (33, 8), (2, 255), (31, 264), (300, 520), (1, 16392), (1000, 40)]


@pytest.mark.parametrize("rows,cols", SHAPES)
def test_quantize(gpu, rows, cols):
    x = spread((rows, cols), 1)
    q, s = gpu.fp4_quantize(x.cuda())
    assert q.dtype == E2M1 and s.dtype == E8M0
    assert tuple(q.shape) == (rows, (cols + 1) // 2) and tuple(s.shape) == (rows, -(-cols // 32))
    assert same((q, s), ref_quantize(x))
    y = gpu.fp4_dequantize(q, s, cols)
    assert torch.equal(y.cpu(), values64(q.cpu(), s.cpu(), cols).float())
    assert torch.equal(gpu.fp4_dequantize(q, s)[:, :cols], y)
    # a value's rounding: half a step
    v = x.double() / torch.pow(2.0, s.cpu().view(torch.uint8).double() - 127).repeat_interleave(32, 1)[:, :cols]
    half = torch.where(v.abs() > 4, 1.0, torch.where(v.abs() > 2, 0.5, 0.25))
    assert bool(((y.cpu().double() / x.double() * v - v).abs() <= half + 1e-12).all())


@pytest.mark.parametrize("rows,cols", SHAPES + [(4096, 33), (33, 4096), (511, 700)])
def test_quantize_columns(gpu, rows, cols):
    """The transposed view of a row-major matrix, of rows wider than the view, off the
    16-byte boundaries."""
    x = spread((cols, rows), 2).t()
    assert same(gpu.fp4_quantize(x.t().cuda().t()), ref_quantize(x))
    wide = torch.full((cols, rows + 5), NAN)
    wide[:, 3:3 + rows] = x.t()
    assert same(gpu.fp4_quantize(wide.cuda()[:, 3:3 + rows].t()), ref_quantize(x))


@pytest.mark.parametrize("columns", [False, True])
def test_quantize_edges(gpu, columns):
    """Blocks of zeros, magnitudes at both ends of fp32 and on the scale's borders (6
    and the value after it), every tie, infinities and NaN."""
    rows = []
    tiny, big = float(np.finfo(np.float32).tiny), float(np.finfo(np.float32).max)
    for v in (0.0, -0.0, 6.0, float(np.nextafter(np.float32(6), np.float32(9))), 1.0, tiny, 1.4e-45, big, 6 * 2.0 ** -126,
              float(np.nextafter(np.float32(6 * 2.0 ** -126), np.float32(0))), 3 * 2.0 ** -126, 5.0, 7.0, 8.0, 1e-40):
        r = torch.linspace(-1, 1, 320) * v
        r[7::32] = v
        rows.append(r)
    ties = torch.tensor([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, 6.0])
    ties = torch.cat((ties, -ties))
    for near in (0.0, 1.0, -1.0):  # on the ties and next to them
        rows.append((ties * (1 + near * 2.0 ** -23)).repeat(20).float())
        rows[-1][7::8] = torch.sign(rows[-1][7::8]) * 6
    for bad in (INF, -INF, NAN):
        r = torch.linspace(-3, 3, 320)
        r[100] = bad
        rows.append(r)
    rows.append(torch.full((320,), INF))
    x = torch.stack(rows)
    got = gpu.fp4_quantize(x.t().contiguous().cuda().t() if columns else x.cuda())
    assert same(got, ref_quantize(x))
    for cols in (319, 313):  # the kernel of rows off the boundaries
        assert same(gpu.fp4_quantize(x[:, :cols].cuda()), ref_quantize(x[:, :cols]))
    y = gpu.fp4_dequantize(*got).cpu()
    want = (~torch.isfinite(x)).view(-1, 10, 32).any(2).repeat_interleave(32, 1)
    assert torch.equal(torch.isnan(y), want)


def test_quantize_strided_and_shaped(gpu):
    wide = spread((40, 400), 3).cuda()
    for x in (wide[:, :256], wide[:, 1:257], wide[3:20, 5:134], wide.t()[:300], wide[:1, :200].expand(9, 200), wide[:, ::2],
              wide[:, :1], wide[:1], wide.t()[:1], wide[:, :1].t()):
        assert same(gpu.fp4_quantize(x), ref_quantize(x))
    x3 = spread((6, 7 * 130), 4).view(6, 7, 130)
    q, s = gpu.fp4_quantize(x3.cuda())
    assert tuple(q.shape) == (6, 7, 65) and tuple(s.shape) == (6, 7, 5)
    assert same((q.view(42, 65), s.view(42, 5)), ref_quantize(x3.view(42, 130)))
    assert tuple(gpu.fp4_dequantize(q, s).shape) == (6, 7, 130)
    assert tuple(gpu.fp4_dequantize(q, s, 129).shape) == (6, 7, 129)
    e, es = gpu.fp4_quantize(torch.empty((0, 40), device="cuda"))
    assert tuple(e.shape) == (0, 20) and tuple(es.shape) == (0, 2) and gpu.fp4_dequantize(e, es).shape == (0, 40)
    e, es = gpu.fp4_quantize(torch.empty((3, 0), device="cuda"))
    assert tuple(e.shape) == (3, 0) and tuple(es.shape) == (3, 0) and gpu.fp4_dequantize(e, es).shape == (3, 0)
    v, vs = gpu.fp4_quantize(wide[0])
    assert same((v[None], vs[None]), ref_quantize(wide[:1]))


def test_dequantize_every_code_and_scale(gpu):
    codes = torch.arange(256, dtype=torch.uint8).repeat(256, 1).cuda().view(E2M1)
    scale = torch.arange(256, dtype=torch.uint8).view(256, 1).repeat(1, 16).cuda().view(E8M0)
    want = values64(codes.cpu(), scale.cpu()).float()
    for cols in (512, 511):
        y = gpu.fp4_dequantize(codes, scale, cols).cpu()
        assert torch.equal(torch.isnan(y), torch.isnan(want[:, :cols]))
        ok = ~torch.isnan(y)
        assert torch.equal(y[ok], want[:, :cols][ok])
    out = torch.full((256, 512), 7.0, device="cuda")
    assert gpu.fp4_dequantize(codes, scale, out=out).data_ptr() == out.data_ptr()
    y = gpu.fp4_dequantize(codes[3:, 5:37], scale[3:, :2])  # rows inside a wider matrix
    assert torch.equal(y[:200].cpu(), values64(codes[3:203, 5:37].cpu(), scale[3:203, :2].cpu()).float())


# ------------------------------------------------------------------ product

def check_product(gpu, a, sa, w, sw, bias=None, act=0, out=None):
    A, W = values64(a, sa), values64(w, sw)
    z, S = A @ W.t(), A.abs() @ W.abs().t()
    if bias is not None:
        z, S = z + bias.double(), S + bias.double().abs()
    bound = S * (2.0 ** -19 + (A.shape[1] / 2048 + 2) * 2.0 ** -24)
    ref = (z, torch.relu(z), torch.sigmoid(z), torch.tanh(z))[act]
    if act >= 2:  # slopes at most 1; the function's own few ulp
        bound = bound + 8 * 2.0 ** -24
    c = gpu.fp4_matmul(a, sa, w.t(), sw.t(), bias, act, out=out)
    assert c.dtype == torch.float32
    off = (c.double() - ref).abs()
    assert bool((off <= bound).all()), float((off / bound.clamp(min=1e-300)).max())
    return c


# few rows and many, tiles with every kind of edge, contractions that end inside a
# block, a word of scales, a stage
PRODUCTS = [(1, 1, 2), (1, 128, 128), (1, 4096, 256), (2, 130, 1000), (3, 100, 30), (4, 257, 4096), (5, 257, 16),
            (7, 33, 34), (8, 1000, 520), (9, 64, 96), (16, 512, 130), (17, 300, 384), (33, 64, 640), (48, 700, 2048),
            (64, 1000, 126), (65, 96, 128), (128, 128, 512), (129, 257, 386), (300, 1000, 1000), (520, 260, 2048),
            (513, 1030, 272), (100, 3, 62), (1, 1, 16384), (1000, 1, 64)]


@pytest.mark.parametrize("m,n,k", PRODUCTS)
def test_product(gpu, m, n, k):
    a, sa = operand(m, k, 11)
    w, sw = operand(n, k, 12)
    check_product(gpu, a, sa, w, sw)


# enough tiles for CTA pairs; more tiles than pairs, ragged edges, several promotions
LARGE = [(1537, 2050, 400), (2600, 2100, 1200), (2310, 2000, 130), (1300, 1800, 9000), (2048, 2304, 4608),
         (4200, 1001, 2050)]


@pytest.mark.parametrize("m,n,k", LARGE)
def test_product_large(gpu, m, n, k):
    a, sa = operand(m, k, 23)
    w, sw = operand(n, k, 24)
    bias = torch.randn(n, generator=torch.Generator().manual_seed(10)).cuda()
    big = torch.full((m + 2, n + 6), 3.0, device="cuda")
    check_product(gpu, a, sa, w, sw, bias, 0, out=big[1:m + 1, 2:n + 2])
    mask = torch.ones_like(big, dtype=torch.bool)
    mask[1:m + 1, 2:n + 2] = False
    assert bool((big[mask] == 3.0).all())
    check_product(gpu, a, sa, w, sw, bias, 1)


@pytest.mark.parametrize("m,n,pad", [(5000, 1018, 2), (5000, 1017, 3), (5000, 1016, 4), (2600, 2051, 1), (9500, 1, 3),
                                     (300, 601, 3), (40, 1001, 3), (3, 1001, 3), (1, 4097, 3)])
def test_product_leaves_the_row_padding(gpu, m, n, pad):
    """What lies behind a row of the output stays as it was, behind the last row too."""
    a, sa = operand(m, 200, 34)
    w, sw = operand(n, 200, 35)
    big = torch.full((m * (n + pad) + 64,), 7.0, device="cuda")
    out = big.as_strided((m, n), (n + pad, 1), 0)
    check_product(gpu, a, sa, w, sw, torch.ones(n, device="cuda"), 0, out=out)
    rest = torch.ones_like(big, dtype=torch.bool)
    rest.as_strided((m, n), (n + pad, 1), 0)[:] = False
    assert bool((big[rest] == 7.0).all())


@pytest.mark.parametrize("act", [0, 1, 2, 3])
@pytest.mark.parametrize("m,n,k", [(1, 200, 256), (3, 200, 256), (20, 200, 256), (200, 330, 256), (2600, 2100, 256)])
def test_product_bias_activation(gpu, m, n, k, act):
    a, sa = operand(m, k, 15)
    w, sw = operand(n, k, 16)
    bias = torch.randn(n, generator=torch.Generator().manual_seed(1)).cuda()
    check_product(gpu, a, sa, w, sw, bias, act)


# long contractions and many columns, every way the work is shared out
LONG = [(1, 20000, 4224), (3, 20000, 4224), (20, 19000, 5000), (64, 20000, 6400), (7, 2048, 16500), (30, 1000, 9000),
        (1, 1920, 4100), (2, 1000, 30000), (128, 2048, 9000), (64, 8300, 8192), (4, 8300, 8192), (16, 8300, 8192)]


@pytest.mark.parametrize("m,n,k", LONG)
def test_product_long(gpu, m, n, k):
    a, sa = operand(m, k, 17)
    w, sw = operand(1280, k, 18)
    at = torch.arange(n, device="cuda") % 1280  # the weight's rows over and over
    check_product(gpu, a, sa, w.view(torch.uint8)[at].view(E2M1), sw.view(torch.uint8)[at].view(E8M0))


@pytest.mark.parametrize("m,n,k", [(1, 2048, 16384), (4, 2048, 16384), (16, 2048, 16384), (64, 20000, 8192),
                                   (300, 2048, 8192), (2048, 8192, 1024), (2600, 2100, 16384)])
def test_product_of_one_sign(gpu, m, n, k):
    """Positive operands with a long tail: nothing cancels, and every addition of the
    accumulator truncates the same way, at most 2^-21 of the running sum a step."""
    g = torch.Generator(device="cuda").manual_seed(33)
    a, sa = gpu.fp4_quantize(torch.exp(3 * torch.randn((m, k), device="cuda", generator=g)))
    w, sw = gpu.fp4_quantize(torch.exp(3 * torch.randn((n, k), device="cuda", generator=g)))
    z = values64(a, sa) @ values64(w, sw).t()
    c = gpu.fp4_matmul(a, sa, w.t(), sw.t())
    assert bool(((c.double() - z).abs() <= z * (64 * 2.0 ** -21 + (k / 2048 + 2) * 2.0 ** -24)).all())


@pytest.mark.parametrize("m,n", [(1, 140), (5, 140), (150, 200), (2600, 2100)])
def test_product_scale_range(gpu, m, n):
    """Scales far from 1 that cancel, the smallest byte, and byte 255 (NaN), on every
    path a size takes."""
    g = torch.Generator().manual_seed(11)
    k = 300
    a = torch.randint(0, 256, (m, k // 2), generator=g).to(torch.uint8).cuda().view(E2M1)
    w = torch.randint(0, 256, (n, k // 2), generator=g).to(torch.uint8).cuda().view(E2M1)
    for ea, ew in ((27, 227), (227, 27), (0, 200), (127, 0), (1, 253)):
        sa = torch.full((m, 10), ea, dtype=torch.uint8).cuda().view(E8M0)
        sw = torch.full((n, 10), ew, dtype=torch.uint8).cuda().view(E8M0)
        check_product(gpu, a, sa, w, sw)
    sa = torch.full((m, 10), 127, dtype=torch.uint8).cuda()
    sw = torch.full((n, 10), 127, dtype=torch.uint8).cuda()
    sa[m - 1, 1] = 255
    sw[n - 2, 9] = 255
    c = gpu.fp4_matmul(a, sa.view(E8M0), w.t(), sw.view(E8M0).t())
    want = torch.zeros_like(c, dtype=torch.bool)
    want[m - 1, :] = True
    want[:, n - 2] = True
    assert torch.equal(torch.isnan(c), want)


def test_product_strides_and_bounds(gpu):
    """Operands inside wider buffers at odd offsets, whose other bytes are NaN scales
    and codes; a weight that lies as its transpose."""
    for m, n, k, off in [(150, 140, 300, 3), (9, 200, 256, 16), (200, 260, 128, 0), (1, 100, 62, 1), (4, 90, 4096, 32),
                         (2000, 2100, 320, 5)]:
        wa, _ = operand(m, k + 80, 40)
        ww, _ = operand(n, k + 96, 41)
        a, w = wa[:, off:off + k // 2], ww[:, off:off + k // 2]
        kb = -(-k // 32)
        full = torch.full((max(m, n), kb + 3), 255, dtype=torch.uint8, device="cuda")
        g = torch.Generator(device="cuda").manual_seed(42)
        sa, sw = full[:m].clone(), full[:n].clone()
        sa[:, 1:1 + kb] = torch.randint(120, 130, (m, kb), device="cuda", generator=g, dtype=torch.uint8)
        sw[:, :kb] = torch.randint(120, 130, (n, kb), device="cuda", generator=g, dtype=torch.uint8)
        sa, sw = sa.view(E8M0)[:, 1:1 + kb], sw.view(E8M0)[:, :kb]
        big = torch.full((m + 4, n + 9), 7.0, device="cuda")
        c = check_product(gpu, a, sa, w, sw, out=big[2:2 + m, 4:4 + n])
        mask = torch.ones_like(big, dtype=torch.bool)
        mask[2:2 + m, 4:4 + n] = False
        assert bool((big[mask] == 7.0).all())
        assert torch.equal(gpu.fp4_matmul(a, sa, w.t().contiguous(), sw.view(torch.uint8).t().contiguous().view(E8M0)), c)


def test_product_empty(gpu):
    a, sa = operand(4, 128, 19)
    w, sw = operand(6, 128, 20)
    bias = torch.arange(6.0, device="cuda") - 2
    z = gpu.fp4_matmul(a[:, :0], sa[:, :0], w[:, :0].t(), sw[:, :0].t(), bias, gpu.ACT_RELU)
    assert torch.equal(z, torch.relu(bias).expand(4, 6))
    assert gpu.fp4_matmul(a[:0], sa[:0], w.t(), sw.t()).shape == (0, 6)
    assert gpu.fp4_matmul(a, sa, w[:0].t(), sw[:0].t()).shape == (4, 0)


@pytest.mark.parametrize("m,n,k", [(70001, 32768, 130), (70001, 32770, 130), (64, 33600000, 128), (3, 750000000, 32),
                                   (9, 240000000, 16)])
def test_product_beyond_2_31_elements(gpu, m, n, k):
    a0, sa0 = operand(min(m, 1000), k, 5)
    w0, sw0 = operand(1280, k, 6)

    def repeated(t, rows):
        return t.view(torch.uint8).repeat(-(-rows // t.shape[0]), 1)[:rows].view(t.dtype)

    c = gpu.fp4_matmul(repeated(a0, m), repeated(sa0, m), repeated(w0, n).t(), repeated(sw0, n).t())
    A, W = values64(a0, sa0), values64(w0, sw0)
    z, S = A @ W.t(), A.abs() @ W.abs().t()
    for r in (0, m // 2 // 1000 * 1000, m - m % 1000 if m > 1000 else 0):
        for t in (0, n // 2 // 1280 * 1280, n // 1280 * 1280 - 1280, n - n % 1280):
            got = c[r:r + 1000, t:t + 1280].double()
            off, most = (got - z[:got.shape[0], :got.shape[1]]).abs(), S[:got.shape[0], :got.shape[1]] * 2.0 ** -18
            assert bool((off <= most).all())
    del c
    torch.cuda.empty_cache()


def test_save_beyond_2_31_elements(gpu):
    rows, d = 530000, 4104
    x0 = spread((1000, d), 7).cuda()
    want = ref_quantize(x0)
    x = x0.repeat(530, 1)
    q, s = gpu.fp4_quantize(x)
    for r in (0, 265000, 529000):
        assert same((q[r:r + 1000], s[r:r + 1000]), want)
    y = gpu.fp4_dequantize(q, s, out=x)
    assert torch.equal(y[529000:].cpu(), values64(want[0], want[1]).float())
    del q, s, y
    x0 = spread((4104, 1000), 8).cuda()
    x.view(4104, rows).view(4104, 530, 1000)[:] = x0[:, None]
    want = ref_quantize(x0.t())
    q, s = gpu.fp4_quantize(x.view(4104, rows).t())
    for r in (0, 265000, 529000):
        assert same((q[r:r + 1000], s[r:r + 1000]), want)
    torch.cuda.empty_cache()


# ------------------------------------------------------------------ a training step

@pytest.mark.parametrize("rows,d,n", [(70, 200, 130), (512, 1024, 768), (2100, 1500, 2200)])
def test_block_step(gpu, rows, d, n):
    """Norm, 4-bit Linear, and back with the same product: the input's gradient through
    the weight quantised the other way, the weight's from both transposes, then the
    norm's.  Each stage against float64 on what the stage before left."""
    g = torch.Generator().manual_seed(90)
    x, res = torch.randn((rows, d), generator=g).cuda(), torch.randn((rows, d), generator=g).cuda()
    nw = (1 + 0.1 * torch.randn(d, generator=g)).cuda()
    weight = (torch.randn((n, d), generator=g) * d ** -0.5).cuda()
    grad = torch.randn((rows, n), generator=g).cuda()
    y, h, rstd = gpu.rms_norm_fwd(x, nw, residual=res)
    yq, wq = gpu.fp4_quantize(y), gpu.fp4_quantize(weight)
    Y = values64(*yq)
    # half a step of e2m1 on its coarsest interval, 1 of 4, bounds a value's rounding
    assert float((Y[:, :d] - y.double()).norm() / y.double().norm()) <= 0.25
    check_product(gpu, *yq, *wq)
    check_product(gpu, *gpu.fp4_quantize(grad), *gpu.fp4_quantize(weight.t()))
    dy = gpu.fp4_matmul(*gpu.fp4_quantize(grad), *[t.t() for t in gpu.fp4_quantize(weight.t())])
    dw = check_product(gpu, *gpu.fp4_quantize(grad.t()), *gpu.fp4_quantize(y.t()))
    assert dy.shape[1] >= d and dw.shape[0] == n
    dx, dnw = gpu.rms_norm_backward(h, rstd, dy, nw, grad_sum=x)
    u = h.double() * rstd.double()[:, None]
    t = dy.double() * nw.double()
    want = rstd.double()[:, None] * (t - u * (t * u).mean(1, keepdim=True)) + x.double()
    assert float((dx.double() - want).norm() / want.norm()) <= 1e-6
    assert float((dnw.double() - (dy.double() * u).sum(0)).norm() / dnw.double().norm()) <= 1e-6


# ------------------------------------------------------------------ streams, graphs, threads

def test_side_stream_and_graphs(gpu):
    """On a side stream, then captured twice and the two graphs replayed at the same
    time with other inputs in the captured buffers."""
    for m, n, k in ((1, 300, 512), (40, 256, 1024), (200, 256, 384), (2100, 2304, 512)):
        xs = [spread((m, k), 50 + i, -1.0, 1.0).cuda() for i in range(2)]
        w, sw = operand(n, k, 60)

        def step(x):
            q, s = gpu.fp4_quantize(x)
            t, ts = gpu.fp4_quantize(x.t())
            return (gpu.fp4_matmul(q, s, w.t(), sw.t()), gpu.fp4_dequantize(q, s), t.view(torch.uint8), ts.view(torch.uint8))

        want = [[t.clone() for t in step(x)] for x in xs]
        torch.cuda.synchronize()
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            got = step(xs[0])
        side.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, want[0]))
        graphs, outs, ins = [], [], []
        for i in range(2):
            ins.append(torch.zeros_like(xs[0]))
            g = torch.cuda.CUDAGraph()
            with torch.cuda.graph(g):
                outs.append(step(ins[i]))
            graphs.append(g)
        for i in range(2):
            ins[i].copy_(xs[i])
        torch.cuda.synchronize()
        streams = [torch.cuda.Stream() for _ in range(2)]
        for _ in range(3):
            for g, s in zip(graphs, streams):
                with torch.cuda.stream(s):
                    g.replay()
        torch.cuda.synchronize()
        for i in range(2):
            assert all(torch.equal(a, b) for a, b in zip(outs[i], want[i]))
    assert gpu.get_context(0).device_error() == 0


@pytest.mark.parametrize("sizes", [((2100, 1900, 400), (40, 500, 640)), ((1, 4096, 2048), (4, 1000, 4096))])
def test_two_threads(gpu, sizes):
    def of(m, n, k):
        a, w = operand(m, k, 80), operand(n, k, 81)
        return lambda: (gpu.fp4_matmul(*a, *[t.t() for t in w]),)

    _two_threads(gpu, [of(*s) for s in sizes])


# ------------------------------------------------------------------ refusals

def test_refusals(gpu):
    x = torch.zeros((4, 256), device="cuda")
    q, s = gpu.fp4_quantize(x)
    w, sw = gpu.fp4_quantize(torch.zeros((9, 256), device="cuda"))
    z = torch.zeros((), device="cuda")
    for call in (lambda: gpu.fp4_quantize(x.half()), lambda: gpu.fp4_quantize(x.cpu()), lambda: gpu.fp4_quantize(z),
                 lambda: gpu.fp4_dequantize(x, s), lambda: gpu.fp4_dequantize(q, s[:, :7]),
                 lambda: gpu.fp4_dequantize(q, s.float()), lambda: gpu.fp4_dequantize(q, s.cpu()),
                 lambda: gpu.fp4_dequantize(q, s, 254), lambda: gpu.fp4_dequantize(q, s, 257),
                 lambda: gpu.fp4_dequantize(q, s, -2), lambda: gpu.fp4_dequantize(q.view(torch.uint8), s),
                 lambda: gpu.fp4_dequantize(q, s, out=torch.zeros((4, 255), device="cuda")),
                 lambda: gpu.fp4_matmul(q, s, w, sw), lambda: gpu.fp4_matmul(q, s[:3], w.t(), sw.t()),
                 lambda: gpu.fp4_matmul(q, s, w.t(), sw.t()[:1]), lambda: gpu.fp4_matmul(x, s, w.t(), sw.t()),
                 lambda: gpu.fp4_matmul(q, s, w[:, :127].t(), sw.t()), lambda: gpu.fp4_matmul(q, s, w.t(), sw),
                 lambda: gpu.fp4_matmul(q, s, w.t(), sw.float().t()),
                 lambda: gpu.fp4_matmul(q, s, w.t(), sw.t(), torch.zeros(7, device="cuda")),
                 lambda: gpu.fp4_matmul(q, s, w.t(), sw.t(), out=torch.zeros((4, 8), device="cuda")),
                 lambda: gpu.fp4_matmul(q, s, w.t(), sw.t(), out=torch.zeros((9, 4), device="cuda").t()),
                 lambda: gpu.fp4_matmul(*gpu.fp8_quantize(x), w.t(), sw.t())):
        with pytest.raises(ValueError):
            call()
    with pytest.raises(gpu.RtbError):
        gpu.fp4_matmul(q, s, w.t(), sw.t(), act=9)
