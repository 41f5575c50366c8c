"""8-bit block-scaled tensors on the B200: writing and restoring them, their
product and the weight gradient that reads a checkpoint, against plain
restatements in float64.

Saving is exact arithmetic with one rounding, so its bytes are compared for
equality.  Products are held elementwise to gamma * S, S = sum of |a||b| over the
contraction: the products of e4m3 codes are exact, the tensor core adds four
steps of 32 (MODE fp8) or 8 steps of 16 for each of three terms (weight
gradient) per 128-element block, each step within 2^-21 of the block's S
(truncated alignment of the addends and of the sum), and every block is added
in fp32 (2^-24 of the running sum, at most S).  Where the tensor core applies the
scales itself, 32 or 64 steps run before the addition, each within 2^-24 of the
running sum, on average half of the unit's S: at most the same 2^-19."""
import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

E4M3 = torch.float8_e4m3fn
E8M0 = torch.float8_e8m0fnu


def ref_quantize(x, block_rows):
    """(codes, scale bytes) by the format's definition, on the CPU."""
    x = x.cpu()
    rows, cols = x.shape
    rb, cb = -(-rows // block_rows), -(-cols // 128)
    full = torch.zeros((rb * block_rows, cb * 128))
    full[:rows, :cols] = torch.where(torch.isfinite(x), x, torch.zeros_like(x))
    top = full.abs().view(rb, block_rows, cb, 128).amax(dim=(1, 3)).double().numpy()
    byte = np.full(top.shape, 127, np.int64)
    for i in np.ndindex(top.shape):
        if top[i] > 0:
            b = 1
            while top[i] / 2.0 ** (b - 127) > 448.0:
                b += 1
            byte[i] = b
    byte = torch.from_numpy(byte)
    scale = torch.pow(2.0, byte.double() - 127).repeat_interleave(block_rows, 0)[:rows]
    scale = scale.repeat_interleave(128, 1)[:, :cols]
    y = (x.double() / scale).float()
    y = torch.where(torch.isfinite(y), y, torch.full_like(y, float("nan")))
    return y.to(E4M3), byte.to(torch.uint8)


def values64(q, scale):
    """The float64 values of (q, scale); scale e8m0 or float32."""
    rows, cols = q.shape
    if scale.dtype == E8M0:
        byte = scale.view(torch.uint8).double()
        s = torch.pow(2.0, byte - 127)
        s[byte == 255] = float("nan")
    else:
        s = scale.double()
    if s.shape[0] != rows:
        s = s.repeat_interleave(128, 0)[:rows]
    return q.float().double() * s.repeat_interleave(128, 1)[:, :cols]


def spread(shape, seed, low=-6.0, high=6.0):
    """Normal values with magnitudes spread over a few powers of ten."""
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(shape, generator=g)
    return x * torch.pow(10.0, low + (high - low) * torch.rand((shape[0], 1), generator=g))


def operand(rows, cols, block_rows, seed):
    x = spread((rows, cols), seed, -1.0, 1.0).cuda()
    q, b = ref_quantize(x, block_rows)
    return q.cuda(), b.cuda().view(E8M0)


def same_codes(got, want):
    g, w = got.view(torch.uint8).cpu(), want.view(torch.uint8).cpu()
    nan = (w & 0x7F) == 0x7F
    assert torch.equal(g[~nan], w[~nan])
    assert bool(((g & 0x7F)[nan] == 0x7F).all())


# ------------------------------------------------------------------ save and restore

SHAPES = [(1, 1), (1, 128), (3, 129), (7, 1000), (130, 64), (128, 128), (257, 385), (64, 4096)]


@pytest.mark.parametrize("rows,cols", SHAPES)
@pytest.mark.parametrize("block_rows", [1, 128])
def test_quantize(gpu, rows, cols, block_rows):
    x = spread((rows, cols), 1)
    q, s = gpu.fp8_quantize(x.cuda(), block_rows)
    wq, ws = ref_quantize(x, block_rows)
    assert q.dtype == E4M3 and s.dtype == E8M0 and tuple(s.shape) == tuple(ws.shape)
    assert torch.equal(s.view(torch.uint8).cpu(), ws)
    same_codes(q, wq)
    y = gpu.fp8_dequantize(q, s)
    want = values64(wq, ws.view(E8M0)).float()
    assert torch.equal(y.cpu(), want)
    # a value's rounding: half a step of e4m3, relative above its subnormals
    off = (y.cpu().double() - x.double()).abs()
    step = torch.pow(2.0, ws.double() - 127).repeat_interleave(block_rows, 0)[:rows]
    step = step.repeat_interleave(128, 1)[:, :cols] * 2.0 ** -10
    assert bool((off <= torch.maximum(x.double().abs() * 2.0 ** -4, step)).all())


@pytest.mark.parametrize("block_rows", [1, 128])
def test_quantize_edges(gpu, block_rows):
    """A block of zeros, magnitudes at both ends of fp32 and on the scale's
    borders (448 and the value after it), ties, infinities and NaN."""
    rows = []
    tiny, big = float(np.finfo(np.float32).tiny), float(np.finfo(np.float32).max)
    for v in (0.0, -0.0, 448.0, float(np.nextafter(np.float32(448), np.float32(1e9))), 1.0, tiny,
              1.4e-45, big, 2.0 ** -118, 1.75 * 2.0 ** -118, 240.0, 464.0):
        r = torch.linspace(-1, 1, 300) * v
        r[7] = v
        rows.append(r)
    ties = torch.arange(300).float() * 0.0625 + 1.03125
    rows.append(ties)
    bad = torch.linspace(-3, 3, 300)
    bad[3], bad[150], bad[299] = float("inf"), float("-inf"), float("nan")
    rows.append(bad)
    rows.append(torch.full((300,), float("inf")))
    rows.append(torch.full((300,), float("nan")))
    x = torch.stack(rows)
    q, s = gpu.fp8_quantize(x.cuda(), block_rows)
    wq, ws = ref_quantize(x, block_rows)
    assert torch.equal(s.view(torch.uint8).cpu(), ws)
    same_codes(q, wq)
    y = gpu.fp8_dequantize(q, s).cpu()
    assert torch.equal(torch.isnan(y), ~torch.isfinite(x))


def test_quantize_strided_and_shaped(gpu):
    """Rows of a wider matrix, a base that no 16-byte load fits, a transposed
    and an expanded input, leading dimensions."""
    wide = spread((40, 400), 3).cuda()
    for x in (wide[:, :256], wide[:, 1:257], wide[3:20, 5:134], wide.t()[:300],
              wide[:1, :200].expand(9, 200)):
        q, s = gpu.fp8_quantize(x)
        wq, ws = ref_quantize(x.contiguous(), 1)
        same_codes(q, wq)
        assert torch.equal(s.view(torch.uint8).cpu(), ws)
    x3 = spread((6, 7 * 130), 4).view(6, 7, 130)
    q, s = gpu.fp8_quantize(x3.cuda())
    assert tuple(q.shape) == (6, 7, 130) and tuple(s.shape) == (6, 7, 2)
    same_codes(q.view(42, 130), ref_quantize(x3.view(42, 130), 1)[0])
    assert tuple(gpu.fp8_dequantize(q, s).shape) == (6, 7, 130)
    e, es = gpu.fp8_quantize(torch.empty((0, 40), device="cuda"))
    assert tuple(e.shape) == (0, 40) and tuple(es.shape) == (0, 1)
    assert gpu.fp8_dequantize(e, es).shape == (0, 40)


def test_dequantize_every_code_and_scale(gpu):
    codes = torch.arange(256, dtype=torch.uint8).repeat(256, 1).cuda().view(E4M3)
    scale = torch.arange(256, dtype=torch.uint8).view(256, 1).repeat(1, 2).cuda().view(E8M0)
    y = gpu.fp8_dequantize(codes, scale).cpu()
    want = values64(codes.cpu(), scale.cpu()).float()
    assert torch.equal(torch.isnan(y), torch.isnan(want))
    ok = ~torch.isnan(want)
    assert torch.equal(y[ok], want[ok])


# ------------------------------------------------------------------ product

def check_product(gpu, a, sa, w, sw, bias=None, act=0, trans=True, out=None):
    A, W = values64(a, sa), values64(w, sw)  # W [N, K] (trans) or [K, N]
    Wt = W.t() if trans else W
    z = A @ Wt
    S = A.abs() @ Wt.abs()
    if bias is not None:
        z = z + bias.double()
        S = S + bias.double().abs()
    blocks = -(-a.shape[1] // 128)
    bound = S * (4 * 2.0 ** -21 + (blocks + 2) * 2.0 ** -24)
    ref = (z, torch.relu(z), torch.sigmoid(z), torch.tanh(z))[act]
    if act >= 2:  # slopes at most 1; the function's own few ulp
        bound = bound + 8 * 2.0 ** -24
    c = gpu.fp8_matmul(a, sa, w.t() if trans else w, sw.t() if trans else sw, bias, act, out=out)
    assert c.dtype == torch.float32
    off = (c.double() - ref).abs()
    assert bool((off <= bound).all()), float((off / bound.clamp(min=1e-300)).max())
    return c


PRODUCTS = [(1, 1, 1), (1, 128, 128), (1, 4096, 256), (2, 130, 1000), (5, 257, 16), (16, 512, 129),
            (17, 300, 384), (33, 64, 640), (64, 1000, 130), (65, 96, 127), (128, 128, 512),
            (129, 257, 385), (300, 1000, 1000), (520, 260, 2048), (513, 1030, 272)]


@pytest.mark.parametrize("m,n,k", PRODUCTS)
@pytest.mark.parametrize("ra,rb", [(1, 128), (1, 1), (128, 128)])
def test_product(gpu, m, n, k, ra, rb):
    a, sa = operand(m, k, ra, 11)
    w, sw = operand(n, k, rb, 12)
    check_product(gpu, a, sa, w, sw)


# enough 256-row tiles for CTA pairs; more tiles than pairs, ragged edges, more
# than one promotion unit (K > 1024) and less than one
LARGE = [(1537, 2050, 400), (2600, 2100, 1200), (2310, 2000, 130)]


@pytest.mark.parametrize("m,n,k", LARGE)
@pytest.mark.parametrize("ra,rb", [(1, 128), (1, 1)])
@pytest.mark.parametrize("floats", [False, True])
def test_product_large(gpu, m, n, k, ra, rb, floats):
    a, sa = operand(m, k, ra, 23)
    w, sw = operand(n, k, rb, 24)
    if floats:
        sw = (0.01 + torch.rand(sw.shape, generator=torch.Generator().manual_seed(9))).cuda()
    g = torch.Generator().manual_seed(10)
    bias = torch.randn(n, generator=g).cuda()
    big = torch.full((m + 2, n + 6), 3.0, device="cuda")
    check_product(gpu, a, sa, w, sw, bias, 0, out=big[1:m + 1, 2:n + 2])
    mask = torch.ones_like(big, dtype=torch.bool)
    mask[1:m + 1, 2:n + 2] = False
    assert bool((big[mask] == 3.0).all())
    check_product(gpu, a, sa, w, sw, bias, 1)


@pytest.mark.parametrize("k", [130, 400, 640, 1100])
def test_product_scales_of_consecutive_tiles(gpu, k):
    """More tiles than CTA pairs, a float scale for every column and rows of the
    output that are stored directly: the column scales of a tile's last blocks
    and of the next tile's first ones lie side by side in shared memory.  An odd
    and an even number of four-block groups; the same bits on every call."""
    m, n = 2600, 2101
    g = torch.Generator().manual_seed(27)
    a, sa = operand(m, k, 1, 28)
    w, _ = operand(n, k, 1, 29)
    # scales apart by far more than the bound from column to column and block to block
    sw = torch.pow(2.0, 8 * torch.rand((n, -(-k // 128)), generator=g) - 4).cuda()
    first = check_product(gpu, a, sa, w, sw)
    for _ in range(60):
        assert torch.equal(gpu.fp8_matmul(a, sa, w.t(), sw.t()), first)


# rows of the output with a pitch of whole 16 bytes, their length not
@pytest.mark.parametrize("m,n,pad", [(5000, 1018, 2), (5000, 1017, 3), (5000, 1019, 1), (5000, 1018, 6),
                                     (5000, 1016, 4), (2600, 2051, 1), (9500, 1, 3), (9500, 5, 11),
                                     (300, 601, 3), (40, 1001, 3)])
@pytest.mark.parametrize("floats", [False, True])
def test_product_leaves_the_row_padding(gpu, m, n, pad, floats):
    """What lies behind a row of the output stays as it was, behind the last row too."""
    k = 200
    a, sa = operand(m, k, 1, 34)
    w, sw = operand(n, k, 1, 35)
    if floats:
        sw = torch.pow(2.0, sw.view(torch.uint8).float() - 127)
    big = torch.full((m * (n + pad) + 64,), 7.0, device="cuda")
    out = big.as_strided((m, n), (n + pad, 1), 0)
    check_product(gpu, a, sa, w, sw, torch.ones(n, device="cuda"), 0, out=out)
    rest = torch.ones_like(big, dtype=torch.bool)
    rest.as_strided((m, n), (n + pad, 1), 0)[:] = False
    assert bool((big[rest] == 7.0).all())


# long contractions: more blocks for a CTA than its scale buffers hold, one CTA a
# tile and every size of cluster, a tile more or fewer than run at once
LONG = [(3, 20000, 4224), (20, 19000, 5000), (64, 20000, 6400), (7, 2048, 16500), (30, 1000, 9000),
        (1, 1920, 4100), (128, 2048, 9000), (64, 8300, 8192), (16, 8300, 8192)]


@pytest.mark.parametrize("m,n,k", LONG)
@pytest.mark.parametrize("rb", [128, 1])
def test_product_long(gpu, m, n, k, rb):
    a, sa = operand(m, k, 1, 17)
    w, sw = operand(1280, k, rb, 18)

    def cycled(t, rows):  # the operand's rows over and over
        at = torch.arange(rows, device="cuda") % t.shape[0]
        return t.view(torch.uint8)[at].view(t.dtype)

    check_product(gpu, a, sa, cycled(w, n), cycled(sw, -(-n // rb)))


# every kernel, with as long a chain in the tensor core's accumulator as it makes
@pytest.mark.parametrize("m,n,k", [(1, 2048, 16384), (16, 2048, 16384), (64, 20000, 8192), (300, 2048, 8192),
                                   (2048, 8192, 1024), (2600, 2100, 16384), (8192, 4096, 4096)])
@pytest.mark.parametrize("floats", [False, True])
def test_product_of_one_sign(gpu, m, n, k, floats):
    """Positive operands with a long tail: nothing cancels, and every addition of the
    accumulator truncates the same way.  A step of 32 products is off by at most
    2^-21 of the running sum; float scales promote it every 4 steps, e8m0 scales
    every 64 at most."""
    g = torch.Generator(device="cuda").manual_seed(33)

    def heavy(rows, block_rows):
        return gpu.fp8_quantize(torch.exp(3 * torch.randn((rows, k), device="cuda", generator=g)), block_rows)

    a, sa = heavy(m, 1)
    w, sw = heavy(n, 128)
    z = values64(a, sa) @ values64(w, sw).t()
    if floats:
        sw = torch.pow(2.0, sw.view(torch.uint8).float() - 127)
    c = gpu.fp8_matmul(a, sa, w.t(), sw.t())
    steps = 4 if floats else 64
    assert bool(((c.double() - z).abs() <= z * (steps * 2.0 ** -21 + (k / 128 + 2) * 2.0 ** -24)).all())


@pytest.mark.parametrize("m,n", [(5, 140), (150, 200), (2600, 2100)])
def test_product_scale_range(gpu, m, n):
    """Scales far from 1 that cancel, the smallest byte, and byte 255 (NaN), on
    every path a size takes."""
    g = torch.Generator().manual_seed(11)
    k = 300
    a = torch.randint(0, 120, (m, k), generator=g).to(torch.uint8).cuda().view(E4M3)
    w = torch.randint(0, 120, (n, k), generator=g).to(torch.uint8).cuda().view(E4M3)
    for ea, ew in ((27, 227), (227, 27), (0, 200), (127, 0)):
        sa = torch.full((m, 3), ea, dtype=torch.uint8).cuda().view(E8M0)
        sw = torch.full((n, 3), ew, dtype=torch.uint8).cuda().view(E8M0)
        check_product(gpu, a, sa, w, sw)
    sa = torch.full((m, 3), 127, dtype=torch.uint8).cuda()
    sw = torch.full((n, 3), 127, dtype=torch.uint8).cuda()
    sa[3, 1] = 255
    sw[n - 2, 2] = 255
    c = gpu.fp8_matmul(a, sa.view(E8M0), w.t(), sw.view(E8M0).t())
    want = torch.zeros_like(c, dtype=torch.bool)
    want[3, :] = True
    want[:, n - 2] = True
    assert torch.equal(torch.isnan(c), want)


def test_product_nan_codes_large(gpu):
    a, sa = operand(2600, 300, 1, 25)
    w, sw = operand(2100, 300, 128, 26)
    a.view(torch.uint8)[1300, 299] = 0x7F
    w.view(torch.uint8)[2099, 5] = 0xFF
    c = gpu.fp8_matmul(a, sa, w.t(), sw.t())
    want = torch.zeros_like(c, dtype=torch.bool)
    want[1300, :] = True
    want[:, 2099] = True
    assert torch.equal(torch.isnan(c), want)


@pytest.mark.parametrize("m,n,k", [(1, 200, 300), (40, 128, 256), (130, 300, 500), (300, 700, 384)])
def test_product_row_major_b(gpu, m, n, k):
    """b given as [K, N] row-major with 128 x 128 blocks."""
    a, sa = operand(m, k, 1, 13)
    b, sb = operand(k, n, 128, 14)
    check_product(gpu, a, sa, b, sb, trans=False)


@pytest.mark.parametrize("act", [0, 1, 2, 3])
@pytest.mark.parametrize("m,n,k", [(3, 200, 256), (200, 330, 256)])
def test_product_bias_activation(gpu, m, n, k, act):
    a, sa = operand(m, k, 1, 15)
    w, sw = operand(n, k, 128, 16)
    bias = torch.randn(n, generator=torch.Generator().manual_seed(1)).cuda()
    check_product(gpu, a, sa, w, sw, bias, act)


@pytest.mark.parametrize("fa,fb,rb", [(True, False, 128), (False, True, 128), (True, True, 1)])
@pytest.mark.parametrize("m", [7, 150])
def test_product_float_scales(gpu, fa, fb, rb, m):
    """Scales that are no powers of two, as weights quantised elsewhere have."""
    g = torch.Generator().manual_seed(2)
    a, sa = operand(m, 400, 1, 17)
    w, sw = operand(270, 400, rb, 18)
    if fa:
        sa = (0.01 + torch.rand(sa.shape, generator=g)).cuda()
    if fb:
        sw = (0.01 + torch.rand(sw.shape, generator=g)).cuda()
    check_product(gpu, a, sa, w, sw)


def test_product_strides_and_bounds(gpu):
    """Operands inside wider buffers at odd offsets; the output inside a larger
    one, whose other elements stay as they were."""
    g = torch.Generator().manual_seed(3)
    for m, n, k, off in [(150, 140, 300, 3), (9, 200, 256, 16), (200, 260, 128, 0)]:
        wide_a = torch.randint(0, 120, (m, k + 40), generator=g).to(torch.uint8).cuda().view(E4M3)
        wide_w = torch.randint(0, 120, (n, k + 48), generator=g).to(torch.uint8).cuda().view(E4M3)
        a, w = wide_a[:, off:off + k], wide_w[:, off:off + k]
        kb = -(-k // 128)
        sa = torch.randint(120, 130, (m, kb + 3), generator=g).to(torch.uint8).cuda().view(E8M0)[:, 1:1 + kb]
        sw = torch.randint(120, 130, (-(-n // 128), kb + 1), generator=g).to(torch.uint8).cuda().view(E8M0)[:, :kb]
        big = torch.full((m + 4, n + 9), 7.0, device="cuda")
        check_product(gpu, a, sa, w, sw, out=big[2:2 + m, 4:4 + n])
        mask = torch.ones_like(big, dtype=torch.bool)
        mask[2:2 + m, 4:4 + n] = False
        assert bool((big[mask] == 7.0).all())


def test_product_empty(gpu):
    a, sa = operand(4, 128, 1, 19)
    w, sw = operand(6, 128, 128, 20)
    bias = torch.arange(6.0, device="cuda") - 2
    z = gpu.fp8_matmul(a[:, :0], sa[:, :0], w[:, :0].t(), sw[:, :0].t(), bias, gpu.ACT_RELU)
    assert torch.equal(z, torch.relu(bias).expand(4, 6))
    assert gpu.fp8_matmul(a[:0], sa[:0], w.t(), sw.t()).shape == (0, 6)
    assert gpu.fp8_matmul(a, sa, w[:0].t(), sw[:0].t()).shape == (4, 0)


@pytest.mark.parametrize("m", [3, 200])
def test_product_nan_stays_in_its_row_and_column(gpu, m):
    a, sa = operand(m, 300, 1, 21)
    w, sw = operand(140, 300, 1, 22)
    a.view(torch.uint8)[1, 299] = 0x7F
    w.view(torch.uint8)[139, 5] = 0xFF
    c = gpu.fp8_matmul(a, sa, w.t(), sw.t())
    want = torch.zeros_like(c, dtype=torch.bool)
    want[1, :] = True
    want[:, 139] = True
    assert torch.equal(torch.isnan(c), want)


# ------------------------------------------------------------------ weight gradient

def check_wgrad(gpu, m, n, k, precision, block_rows=1, accumulate=False, seed=31):
    a, sa = operand(m, k, block_rows, seed)
    grad = spread((m, n), seed + 1, -4.0, -2.0).cuda()
    A = values64(a, sa)
    ref, S = A.t() @ grad.double(), A.abs().t() @ grad.double().abs()
    # 8 steps for each of the terms; two terms keep 16 bits of the gradient
    terms = 3 if precision == 0 else 2
    bound = S * (8 * terms * 2.0 ** -21 + (-(-m // 128) + 2) * 2.0 ** -24)
    if terms == 2:
        bound = bound + S * 2.0 ** -16
    out = None
    if accumulate:
        out = torch.randn((k, n), generator=torch.Generator().manual_seed(5)).cuda()
        ref = ref + out.double()
        bound = bound + out.double().abs() * 2.0 ** -23
    da, db = gpu.matmul_backward_fp8(a, sa, None, grad, need_a=False, out_b=out,
                                     accumulate=accumulate, precision=precision)
    assert da is None and tuple(db.shape) == (k, n)
    off = (db.double() - ref).abs()
    assert bool((off <= bound).all()), float((off / bound.clamp(min=1e-300)).max())


@pytest.mark.parametrize("m,n,k", [(1, 1, 1), (1, 130, 257), (3, 64, 100), (64, 128, 128),
                                   (65, 100, 7), (127, 256, 130), (129, 300, 385), (515, 260, 136),
                                   (1000, 129, 640), (2050, 520, 264)])
@pytest.mark.parametrize("precision", [0, 1])
def test_weight_gradient(gpu, m, n, k, precision):
    check_wgrad(gpu, m, n, k, precision)


@pytest.mark.parametrize("m,n,k", [(300, 2050, 1537), (1100, 2100, 2600)])
def test_weight_gradient_large(gpu, m, n, k):
    check_wgrad(gpu, m, n, k, 0)
    check_wgrad(gpu, m, n, k, 0, accumulate=True)


def test_weight_gradient_accumulates(gpu):
    check_wgrad(gpu, 200, 150, 260, 0, accumulate=True)
    check_wgrad(gpu, 200, 150, 260, 0, block_rows=128)


def test_matmul_backward_both(gpu):
    a, sa = operand(150, 140, 1, 41)
    b = torch.randn((140, 90), generator=torch.Generator().manual_seed(6)).cuda()
    grad = torch.randn((150, 90), generator=torch.Generator().manual_seed(7)).cuda()
    da, db = gpu.matmul_backward_fp8(a, sa, b, grad)
    A = values64(a, sa)
    for got, ref in ((da, grad.double() @ b.double().t()), (db, A.t() @ grad.double())):
        assert float((got.double() - ref).norm() / ref.norm()) <= 1e-5


def test_weight_gradient_empty_and_special(gpu):
    a, sa = operand(0 + 5, 130, 1, 42)
    z = gpu.matmul_backward_fp8(a[:0], sa[:0], None, torch.empty((0, 9), device="cuda"),
                                need_a=False)[1]
    assert torch.equal(z, torch.zeros((130, 9), device="cuda"))
    keep = torch.ones((130, 9), device="cuda")
    gpu.matmul_backward_fp8(a[:0], sa[:0], None, torch.empty((0, 9), device="cuda"), need_a=False,
                            out_b=keep, accumulate=True)
    assert bool((keep == 1).all())
    # a NaN in the checkpoint or the gradient reaches its row or column alone;
    # an infinite gradient is infinite where the checkpoint is not zero
    a.view(torch.uint8)[2, 7] = 0x7F
    a.view(torch.uint8)[3, 8:] = 0x38  # 1.0
    grad = torch.ones((5, 40), device="cuda")
    grad[3, 11] = float("inf")
    db = gpu.matmul_backward_fp8(a, sa, None, grad, need_a=False)[1]
    assert bool(torch.isnan(db[7]).all())
    assert bool(torch.isinf(db[8:, 11]).all())
    rest = torch.ones_like(db, dtype=torch.bool)
    rest[7, :] = False
    rest[:, 11] = False
    assert bool(torch.isfinite(db[rest]).all())


@pytest.mark.parametrize("precision", [0, 1])
def test_weight_gradient_range(gpu, precision):
    """Gradients at both ends of fp32: its largest value stays finite (bf16's is
    smaller), small normal ones keep their bits."""
    a = torch.full((3, 8), 0x38, dtype=torch.uint8).cuda().view(E4M3)  # 1.0
    sa = torch.full((3, 1), 126, dtype=torch.uint8).cuda().view(E8M0)  # 1/2
    grad = torch.zeros((3, 16), device="cuda")
    grad[1, 0] = float(np.finfo(np.float32).max)
    grad[1, 1] = -float(np.finfo(np.float32).max)
    grad[2, 2] = 1.2345678e-30
    db = gpu.matmul_backward_fp8(a, sa, None, grad, need_a=False, precision=precision)[1]
    want = 0.5 * grad.double().sum(0)
    # 24 bits (TF32 mode: 16); the third term of 1e-30 is a normal bf16
    tol = 2.0 ** -22 if precision == 0 else 2.0 ** -16
    assert bool(((db.double() - want).abs() <= tol * want.abs()).all())


def test_expanded_gradient(gpu):
    """The gradient of a sum arrives as one value expanded over the matrix."""
    a, sa = operand(70, 140, 1, 43)
    grad = torch.ones((), device="cuda").expand(70, 33)
    db = gpu.matmul_backward_fp8(a, sa, None, grad, need_a=False)[1]
    ref = values64(a, sa).sum(0)[:, None].expand(140, 33)
    S = values64(a, sa).abs().sum(0)[:, None]
    assert bool(((db.double() - ref).abs() <= S * 2.0 ** -16).all())


# ------------------------------------------------------------------ streams and graphs

def test_side_stream_and_graphs(gpu):
    """The whole step on a side stream, then captured twice and the two graphs
    replayed at the same time with other inputs in the captured buffers."""
    m, n, k = 200, 256, 384
    xs = [spread((m, k), 50 + i, -1.0, 1.0).cuda() for i in range(2)]
    w, sw = operand(n, k, 128, 60)
    grads = [spread((m, n), 70 + i, -1.0, 1.0).cuda() for i in range(2)]

    def step(x, grad):
        q, s = gpu.fp8_quantize(x)
        y = gpu.fp8_matmul(q, s, w.t(), sw.t())
        return y, gpu.matmul_backward_fp8(q, s, None, grad, need_a=False)[1], gpu.fp8_dequantize(q, s)

    want = [[t.clone() for t in step(x, g)] for x, g in zip(xs, grads)]
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = step(xs[0], grads[0])
    side.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want[0]))

    graphs, outs, ins = [], [], []
    for i in range(2):
        xi, gi = torch.zeros_like(xs[0]), torch.zeros_like(grads[0])
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(step(xi, gi))
        graphs.append(g)
        ins.append((xi, gi))
    for i in range(2):
        ins[i][0].copy_(xs[i])
        ins[i][1].copy_(grads[i])
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


def test_two_threads(gpu):
    """Two host threads, a stream each, the same context."""
    import threading
    a, sa = operand(2100, 400, 1, 80)
    w, sw = operand(1900, 400, 128, 81)
    b, sb = operand(40, 640, 1, 82)
    v, sv = operand(500, 640, 1, 83)
    want = [gpu.fp8_matmul(a, sa, w.t(), sw.t()), gpu.fp8_matmul(b, sb, v.t(), sv.t())]
    torch.cuda.synchronize()
    got, streams = [[], []], [torch.cuda.Stream(), torch.cuda.Stream()]

    def work(i, args):
        with torch.cuda.stream(streams[i]):
            for _ in range(20):
                got[i].append(gpu.fp8_matmul(*args))

    ts = [threading.Thread(target=work, args=(0, (a, sa, w.t(), sw.t()))),
          threading.Thread(target=work, args=(1, (b, sb, v.t(), sv.t())))]
    for t in ts:
        t.start()
    for t in ts:
        t.join()
    torch.cuda.synchronize()
    for i in range(2):
        assert len(got[i]) == 20 and all(torch.equal(c, want[i]) for c in got[i])


# ------------------------------------------------------------------ a training step

@pytest.mark.parametrize("rows,d,n", [(70, 200, 130), (512, 1024, 768)])
def test_block_step(gpu, rows, d, n):
    """Layer norm, save, 8-bit Linear with ReLU, and back: the weight gradient
    out of the saved operand, the input's gradient through the weight and the
    norm, whose own input was saved too.  Each stage against float64 on what the
    stage before left."""
    g = torch.Generator().manual_seed(90)
    x = (torch.randn((rows, d), generator=g) + 0.3).cuda()
    nw, nb = (1 + 0.1 * torch.randn(d, generator=g)).cuda(), (0.1 * torch.randn(d, generator=g)).cuda()
    weight = (torch.randn((n, d), generator=g) * d ** -0.5).cuda()
    bias = (0.1 * torch.randn(n, generator=g)).cuda()
    grad = torch.randn((rows, n), generator=g).cuda()

    xq, xs = gpu.fp8_quantize(x)
    y, mean, rstd = gpu.layer_norm_fwd(x, nw, nb)
    yq, ys = gpu.fp8_quantize(y)
    wq, ws = gpu.fp8_quantize(weight, 128)
    z = gpu.fp8_matmul(yq, ys, wq.t(), ws.t(), bias, gpu.ACT_RELU)
    Y, W = values64(yq, ys), values64(wq, ws)
    pre = Y @ W.t() + bias.double()
    S = Y.abs() @ W.abs().t() + bias.double().abs()
    assert bool(((z.double() - torch.relu(pre)).abs() <= S * 2.0 ** -18).all())
    # the saved operand stands for y within half a step of e4m3
    assert float((Y - y.double()).norm() / y.double().norm()) <= 2.0 ** -4

    dz = grad * (z > 0)
    wd = gpu.fp8_dequantize(wq, ws)
    dy, dw = gpu.matmul_backward_fp8(yq, ys, wd.t().contiguous(), dz)
    assert float((dw.double() - Y.t() @ dz.double()).norm() / dw.double().norm()) <= 1e-6
    assert float((dy.double() - dz.double() @ W).norm() / dy.double().norm()) <= 1e-5
    dx, dg, db = gpu.layer_norm_backward(xq, mean, rstd, dy, nw, nb, x_scale=xs)
    u = (values64(xq, xs) - mean.double()[:, None]) * rstd.double()[:, None]
    h = dy.double() * nw.double()
    ref = rstd.double()[:, None] * (h - h.mean(1, keepdim=True) - u * (h * u).mean(1, keepdim=True))
    for got, want in ((dx, ref), (dg, (dy.double() * u).sum(0)), (db, dy.double().sum(0))):
        assert float((got.double() - want).norm() / want.norm()) <= 1e-6
    # gradients through the checkpoint point where the exact ones do
    u = (x.double() - mean.double()[:, None]) * rstd.double()[:, None]
    ref = rstd.double()[:, None] * (h - h.mean(1, keepdim=True) - u * (h * u).mean(1, keepdim=True))
    assert float((dx.double() - ref).norm() / ref.norm()) <= 2.0 ** -4


# ------------------------------------------------------------------ refusals

def test_refusals(gpu):
    x = torch.zeros((4, 256), device="cuda")
    q, s = gpu.fp8_quantize(x)
    w, sw = gpu.fp8_quantize(torch.zeros((8, 256), device="cuda"), 128)
    for call in (lambda: gpu.fp8_quantize(x.half()),
                 lambda: gpu.fp8_quantize(x, 64),
                 lambda: gpu.fp8_quantize(x.view(2, 2, 256), 128),
                 lambda: gpu.fp8_quantize(x.cpu()),
                 lambda: gpu.fp8_dequantize(x, s),
                 lambda: gpu.fp8_dequantize(q, s[:, :1]),
                 lambda: gpu.fp8_dequantize(q, s.float()),
                 lambda: gpu.fp8_dequantize(q, s.cpu()),
                 lambda: gpu.fp8_matmul(q, s, w, sw),
                 lambda: gpu.fp8_matmul(q, s[:3], w.t(), sw.t()),
                 lambda: gpu.fp8_matmul(q, s, w.t(), sw.t()[:1]),
                 lambda: gpu.fp8_matmul(x, s, w.t(), sw.t()),
                 lambda: gpu.fp8_matmul(q, s, w.t(), sw.t(), torch.zeros(7, device="cuda")),
                 lambda: gpu.fp8_matmul(q, s, w.t(), sw.t(), out=torch.zeros((4, 9), device="cuda")),
                 lambda: gpu.fp8_matmul(q, s, q.t().contiguous(), s.t().contiguous()),
                 lambda: gpu.matmul_backward_fp8(q, s, None, x),
                 lambda: gpu.matmul_backward_fp8(q, s, None, x[:3], need_a=False),
                 lambda: gpu.matmul_backward_fp8(q, s.float(), None, x, need_a=False),
                 lambda: gpu.matmul_backward_fp8(q, s, None, x, need_a=False, accumulate=True),
                 lambda: gpu.matmul_backward_fp8(q, s, x, x)):
        with pytest.raises(ValueError):
            call()
    with pytest.raises(gpu.RtbError):
        gpu.fp8_matmul(q, s, w.t(), sw.t(), act=9)
    with pytest.raises(gpu.RtbError):
        gpu.matmul_backward_fp8(q, s, None, x, need_a=False, precision=7)
