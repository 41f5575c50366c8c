"""Block-scaled products whose output fills a part of a tile only, summed over a cluster of
CTAs: most of its CTAs own rows, or columns, of padding, load nothing of the others' and
are done ahead of them.

With scales of 1 every product of codes is a multiple of 1/4 (4 bits) or a small whole
number (8 bits) and every sum is far below 2^22: exact in any order, so that the results
are compared for equality, each call's of a row of calls that run into one another."""
import pytest
import torch

pytestmark = pytest.mark.gpu

E2M1, E4M3, E8M0 = torch.float4_e2m1fn_x2, torch.float8_e4m3fn, torch.float8_e8m0fnu

# one row, few rows and few columns, of tiles of 16, 32, 64 and 128; 1, 2, 4 and 8 parts
SIZES = [(1, 8192, 16384), (1, 130, 16384), (5, 130, 8192), (6, 1, 16384), (9, 4096, 4096), (17, 200, 8192), (31, 4, 4096),
         (33, 130, 16384), (64, 129, 4096), (65, 3, 4096), (100, 65, 8192), (129, 129, 8192), (200, 1, 2048)]


def scales(rows, blocks):
    return torch.full((rows, blocks), 127, dtype=torch.uint8, device="cuda").view(E8M0)


@pytest.mark.parametrize("m,n,k", SIZES)
def test_padding_beside_a_cluster(gpu, m, n, k):
    g = torch.Generator(device="cuda").manual_seed(91)
    grid = torch.tensor([0, 0.5, 1, 1.5, 2, 3, 4, 6, 0, -0.5, -1, -1.5, -2, -3, -4, -6], dtype=torch.float64, device="cuda")
    codes = [torch.randint(0, 16, (r, k), device="cuda", generator=g, dtype=torch.uint8) for r in (m, n)]
    packed = [(c[:, 0::2] | (c[:, 1::2] << 4)).view(E2M1) for c in codes]
    a, w = (grid[c.long()] for c in codes)
    bias = torch.arange(n, device="cuda").float()
    want4 = a @ w.t() + bias
    sa, sw = scales(m, -(-k // 32)), scales(n, -(-k // 32))
    small = [torch.randint(-4, 5, (r, k), device="cuda", generator=g) for r in (m, n)]
    want8 = small[0].double() @ small[1].double().t() + bias
    eight = [t.float().to(E4M3) for t in small]
    sa8, sw8 = scales(m, -(-k // 128)), scales(n, -(-k // 128))
    got = []
    for _ in range(20):
        got.append(gpu.fp4_matmul(packed[0], sa, packed[1].t(), sw.t(), bias))
        got.append(gpu.fp8_matmul(eight[0], sa8, eight[1].t(), sw8.t(), bias))
    for c4, c8 in zip(got[0::2], got[1::2]):
        assert torch.equal(c4.double(), want4) and torch.equal(c8.double(), want8)
    assert gpu.get_context(0).device_error() == 0
