"""The root-mean-square norm and the 4-bit calls where they meet the rest: tensors with
no memory of their own, few rows with rows that begin at any byte, graphs whose products
copy their operands, outputs that no view can describe."""
import os
import subprocess
import sys

import pytest
import torch

from test_fp4_gpu import E2M1, E8M0, check_product, operand, same, spread, ref_quantize

pytestmark = pytest.mark.gpu

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))

PROGRAM = """
import torch
import rustorch_b200 as rb
x = torch.zeros((3, 4, 256), device="cuda")
q, s = rb.fp4_quantize(x)
p, t = rb.fp8_quantize(x)
m = torch.zeros((3, 4), device="cuda")
torch.cuda.synchronize()
calls = (lambda X, Q, S, P, T, M: rb.rms_norm_fwd(X, residual=X),
         lambda X, Q, S, P, T, M: rb.rms_norm_fp8(X),
         lambda X, Q, S, P, T, M: rb.rms_norm_backward(X, M, X, grad_sum=X),
         lambda X, Q, S, P, T, M: rb.rms_norm_backward(P, M, X, x_scale=T),
         lambda X, Q, S, P, T, M: rb.fp4_quantize(X),
         lambda X, Q, S, P, T, M: rb.fp4_dequantize(Q, S),
         lambda X, Q, S, P, T, M: rb.fp4_matmul(Q, S, Q.t(), S.t()))
for call in calls:
    try:
        torch.vmap(call)(x, q, s, p, t, m)
    except (RuntimeError, ValueError) as e:
        print("refused:", str(e).splitlines()[0])
    else:
        raise AssertionError("not refused")
    assert torch.equal(rb.fp4_dequantize(*rb.fp4_quantize(x)), x)  # the next call is as usual
print("fine")
"""


def test_a_transforms_tensors(gpu):
    """torch.vmap's tensors have no data pointer: asking for it throws in the middle of a
    call, which ends as an exception and does not end the process."""
    r = subprocess.run([sys.executable, "-c", PROGRAM], cwd=ROOT, capture_output=True, text=True,
                       timeout=240)
    assert r.returncode == 0 and "fine" in r.stdout, (r.returncode, r.stdout, r.stderr[-2000:])


def placed(t, offset, pad):
    """t's rows `pad` bytes apart, the first at byte `offset`, NaN scales' bytes around."""
    b = t.view(torch.uint8)
    rows, d = b.shape
    wide = torch.full((offset + rows * (d + pad) + 64,), 255, dtype=torch.uint8, device="cuda")
    v = wide.as_strided((rows, d), (d + pad, 1), offset)
    v.copy_(b)
    return v.view(t.dtype)


@pytest.mark.parametrize("offset", range(16))
@pytest.mark.parametrize("m", [1, 2, 3, 4])
def test_few_rows_at_every_byte(gpu, m, offset):
    """Rows of every length modulo a word and a block, at every byte of 16."""
    for n, k, pad in ((1, 64, 0), (5, 2, 1), (6, 30, 2), (33, 34, 5), (64, 1000 + 2 * offset, 0), (9, 2046, 16 - offset)):
        a, sa = operand(m, k, 70 + offset)
        w, sw = operand(n, k, 71 + offset)
        check_product(gpu, placed(a, 15 - offset, pad), placed(sa, offset, pad), placed(w, offset, pad),
                      placed(sw, 15 - offset, pad))


@pytest.mark.parametrize("m,n,k", [(1, 64, 40002), (1, 64, 40000), (1, 1, 32800), (2, 5, 33000), (3, 100, 10010),
                                   (4, 33, 9000), (4, 4096, 9002), (2, 12000, 16392), (1, 5000, 32770)])
@pytest.mark.parametrize("offset", [0, 3])
def test_few_rows_longer_than_what_is_kept_of_them(gpu, m, n, k, offset):
    """Contractions laid out a piece at a time, shared by 1 to 8 warps."""
    a, sa = operand(m, k, 72)
    w, sw = operand(n, k, 73)
    check_product(gpu, a, sa, placed(w, offset, offset), placed(sw, offset, 0))


@pytest.mark.parametrize("m,n,k", [(3, 1001, 1002), (40, 515, 1002), (300, 700, 330), (2100, 2304, 300), (2100, 2303, 514)])
def test_products_that_copy_their_operands(gpu, m, n, k):
    """On a side stream, then captured twice and both replayed at once: rows that the
    tensor cores' loads cannot take are copied into each graph's own workspace."""
    w, sw = operand(n, k, 75)
    xs = [spread((m, k), 76 + i, -1.0, 1.0).cuda() for i in range(2)]
    out = [torch.empty((m, n), device="cuda") for _ in range(2)]

    def step(x, y):
        q, s = gpu.fp4_quantize(x)
        return gpu.fp4_matmul(q, s, w.t(), sw.t(), out=y)

    want = [step(x, torch.empty((m, n), device="cuda")) for x in xs]
    q, s = gpu.fp4_quantize(xs[0])
    assert torch.equal(check_product(gpu, q, s, w, sw), want[0])
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = step(xs[1], torch.empty((m, n), device="cuda"))
    side.synchronize()
    assert torch.equal(got, want[1])
    graphs, ins = [], []
    for i in range(2):
        ins.append(torch.zeros_like(xs[0]))
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            step(ins[i], out[i])
        graphs.append(g)
    streams = [torch.cuda.Stream() for _ in range(2)]
    for turn in range(3):
        for i in range(2):
            ins[i].copy_(xs[(i + turn) % 2])
        torch.cuda.synchronize()
        for g, st in zip(graphs, streams):
            with torch.cuda.stream(st):
                g.replay()
        torch.cuda.synchronize()
        for i in range(2):
            assert torch.equal(out[i], want[(i + turn) % 2])
    assert gpu.get_context(0).device_error() == 0


def test_norm_into_what_no_view_describes(gpu):
    """Leading dimensions that do not fold into one stride, as inputs and as outputs."""
    x = torch.randn((6, 5, 40), generator=torch.Generator().manual_seed(1)).cuda()
    y, h, rstd = gpu.rms_norm_fwd(x, residual=x)
    turned = x.transpose(0, 1)
    assert torch.equal(gpu.rms_norm_fwd(turned, residual=turned)[0], y.transpose(0, 1))
    assert torch.equal(gpu.rms_norm_fwd(turned.contiguous(), residual=turned)[2], rstd.t())
    for k in ("out", "out_sum"):
        with pytest.raises((ValueError, RuntimeError)):
            gpu.rms_norm_fwd(x, residual=x, **{k: torch.empty((5, 6, 40), device="cuda").transpose(0, 1)})
        with pytest.raises(ValueError):
            gpu.rms_norm_fwd(x, residual=x, **{k: torch.empty((6, 40), device="cuda")[:, None].expand(6, 5, 40)[..., ::2]})
    one = torch.zeros((1, 1, 40), device="cuda").expand(6, 5, 40)
    with pytest.raises((ValueError, RuntimeError)):
        gpu.rms_norm_fwd(x, out=one)
    assert torch.equal(gpu.rms_norm_fwd(x, residual=x)[0], y)


def test_save_of_turned_and_sliced_views(gpu):
    """Views whose leading dimensions do not fold, every other column, one repeated row."""
    x = spread((210, 70), 3).view(6, 35, 70).cuda()
    for v in (x.transpose(0, 1), x[:, :, ::2], x[:, 0].t(), x[0].expand(4, 35, 70), x[:, 3:4, 1:34], x[::2]):
        q, s = gpu.fp4_quantize(v)
        cols = v.shape[-1]
        flat = v.reshape(-1, cols)
        assert q.shape == v.shape[:-1] + ((cols + 1) // 2,) and s.shape == v.shape[:-1] + (-(-cols // 32),)
        assert same((q.view(torch.uint8).reshape(flat.shape[0], -1).view(E2M1),
                     s.view(torch.uint8).reshape(flat.shape[0], -1).view(E8M0)), ref_quantize(flat))
        if q.dim() == 3:
            assert torch.equal(gpu.fp4_dequantize(q.transpose(0, 1), s.transpose(0, 1), cols),
                               gpu.fp4_dequantize(q, s, cols).transpose(0, 1))
