"""4-bit products with scales far apart.

First, ones whose two scales multiply to more or less than fp32 holds, on every path
that a size takes: the result is finite where the product of a block's sum and both scales
is.  One block's few products are exact in any order, so that results are compared for
equality with the float64 value rounded once (each is a number of fp32, or 0).

Then whole rows whose blocks' scales lie far apart: on the tensor cores an addition of 64
products truncates by at most 2^-21 of the sum so far, which leaves the accumulator after 64
of them at most and is added up in fp32: (64 2^-21 + (K / 1024 + 2) 2^-24) S, S = sum of |a||b|."""
import pytest
import torch

pytestmark = pytest.mark.gpu

E2M1, E8M0 = torch.float4_e2m1fn_x2, torch.float8_e8m0fnu
GRID = [0, 0.5, 1, 1.5, 2, 3, 4, 6, 0, -0.5, -1, -1.5, -2, -3, -4, -6]


def packed(rows, k, first):
    code = torch.zeros((rows, k), dtype=torch.uint8, device="cuda")
    code[:, :len(first)] = torch.tensor(first, dtype=torch.uint8, device="cuda")
    return (code[:, 0::2] | (code[:, 1::2] << 4)).view(E2M1)


# codes of a row of A and of the weight, the two scale bytes: zeros and sums that cancel
# beside the largest scales, the smallest product beside scales whose product is 2^128 and
# 2^129, ordinary numbers and subnormal ones out of scales far apart
CASES = [([0], [0], 254, 254), ([2, 2], [2, 10], 254, 254), ([7, 7, 5], [7, 15, 0], 250, 140), ([1], [1], 227, 155),
         ([1], [1], 155, 227), ([1, 9], [1, 1], 254, 254), ([1], [9], 192, 191), ([2], [2], 254, 0), ([2], [2], 0, 254),
         ([7, 5], [7, 5], 220, 30), ([2], [2], 57, 57), ([4], [4], 0, 107), ([4], [12], 107, 0), ([4], [4], 0, 0)]


@pytest.mark.parametrize("m,n,k", [(1, 140, 64), (2, 140, 96), (3, 141, 32), (4, 140, 2048), (1, 140, 70), (5, 140, 64),
                                   (30, 140, 96), (60, 140, 64), (150, 200, 64), (300, 300, 4096), (2600, 2100, 64)])
def test_scales_beyond_fp32(gpu, m, n, k):
    grid = torch.tensor(GRID, dtype=torch.float64)
    for a, w, ea, ew in CASES:
        total = float((grid[a] * grid[w]).sum()) * 2.0 ** (ea + ew - 254)
        s = [torch.full((r, -(-k // 32)), e, dtype=torch.uint8, device="cuda").view(E8M0) for r, e in ((m, ea), (n, ew))]
        c = gpu.fp4_matmul(packed(m, k, a), s[0], packed(n, k, w).t(), s[1].t())
        want = torch.tensor(total, dtype=torch.float64).float()
        assert bool((c == want.cuda()).all()), (a, w, ea, ew, total, c[0, 0].item())


@pytest.mark.parametrize("m,n", [(1, 140), (4, 140), (5, 140), (150, 200), (2600, 2100)])
def test_nan_scale_beside_any_other(gpu, m, n):
    for other in (0, 1, 127, 254, 255):
        for ea, ew in ((255, other), (other, 255)):
            s = [torch.full((r, 2), e, dtype=torch.uint8, device="cuda").view(E8M0) for r, e in ((m, ea), (n, ew))]
            assert bool(torch.isnan(gpu.fp4_matmul(packed(m, 64, [2]), s[0], packed(n, 64, [2]).t(), s[1].t())).all())


@pytest.mark.parametrize("m,n,k", [(2, 1000, 4096), (16, 2048, 4096), (300, 2048, 2048), (2600, 2100, 4096), (1500, 2500, 5002)])
@pytest.mark.parametrize("apart", [4, 18, 30, 60])
@pytest.mark.parametrize("signs", [0xFF, 0x77])
def test_scales_apart(gpu, m, n, k, apart, signs):
    g = torch.Generator(device="cuda").manual_seed(92)
    grid = torch.tensor(GRID, dtype=torch.float64, device="cuda")

    def operand(rows):
        byte = torch.randint(0, 256, (rows, k // 2), device="cuda", generator=g, dtype=torch.uint8) & signs
        scale = torch.randint(127 - apart // 2, 128 + apart // 2, (rows, -(-k // 32)), device="cuda", generator=g,
                              dtype=torch.uint8)
        value = torch.stack((grid[(byte & 15).long()], grid[(byte >> 4).long()]), 2).view(rows, k)
        value *= torch.pow(2.0, scale.double() - 127).repeat_interleave(32, 1)[:, :k]
        return byte.view(E2M1), scale.view(E8M0), value

    a, sa, A = operand(m)
    w, sw, W = operand(n)
    c = gpu.fp4_matmul(a, sa, w.t(), sw.t())
    bound = (64 * 2.0 ** -21 + (k / 1024 + 2) * 2.0 ** -24) * (A.abs() @ W.abs().t())
    assert bool(((c.double() - A @ W.t()).abs() <= bound).all())
