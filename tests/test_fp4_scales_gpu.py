"""4-bit products whose two scales multiply to more or less than fp32 holds, on every path
that a size takes: the result is finite where the product of a block's sum and both scales
is.  One block's few products are exact in any order, so that results are compared for
equality with the float64 value rounded once (each is a number of fp32, or 0)."""
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
