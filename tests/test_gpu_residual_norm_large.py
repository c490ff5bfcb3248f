"""Residual addition and norm of rows whose numbers are near the end of fp32's range, or of bf16's: as long as they are finite, and
their products with the weights, so are scales and codes.  Definition and bounds are those of test_gpu_residual_norm."""

import pytest
import torch

from test_gpu_residual_norm import DEV, TYPES, call, check

pytestmark = pytest.mark.gpu

WIDTHS = [8, 100, 128, 1000, 1024, 2050, 4095, 4096, 8191, 9001, 12288, 16384, 20001, 32768]


def rows(W, dtype, g):
    """Small numbers; one, three and all that are large; all of the same; numbers of every size."""
    x = torch.randn(7, W, generator=g)
    x[1, W // 2] = 2e38
    x[2, torch.randperm(W, generator=g)[:3]] = -2e38
    x[3] = 3e38 * torch.sign(x[3])
    x[4] = x[4] * 1e30
    x[5] = 2.5e38
    x[6] *= 10.0 ** (torch.rand(W, generator=g) * 38)
    return x.clamp(-3e38, 3e38).to(dtype)


@pytest.mark.parametrize("grouped", [False, True])
@pytest.mark.parametrize("dtype", ["bf16", "fp32"])
@pytest.mark.parametrize("W", WIDTHS)
def test_large_numbers(W, dtype, grouped):
    g = torch.Generator().manual_seed(W)
    x = rows(W, TYPES[dtype], g).to(DEV)
    w = (0.25 + 0.75 * torch.rand(W, generator=g)).to(TYPES[dtype]).to(DEV)
    codes, scale = call(x, None, w, grouped)
    check(x, None, w, grouped, codes, scale)


@pytest.mark.parametrize("grouped", [False, True])
@pytest.mark.parametrize("W", [512, 999])
def test_sums_and_products_beyond_the_range(W, grouped):
    """Sums of x and the residual are fp32's, as are products with the weights: what passes it makes the row NaN, and no other."""
    g = torch.Generator().manual_seed(W)
    x, r = (rows(W, torch.float32, g).to(DEV) * 0.5 for _ in range(2))
    w = torch.ones(W, device=DEV)
    before, out = r.clone(), torch.zeros_like(r)
    codes, scale = call(x, r, w, grouped, r_out=out)
    check(x, before, w, grouped, codes, scale)
    x[2], r[2] = 3e38, 3e38
    w[3], x[:, 3], r[:, 3] = 2.0, 0.0, 0.0
    x[5, 3] = 2e38
    codes, scale = call(x, r, w, grouped, r_out=out)
    bad = torch.tensor([i in (2, 5) for i in range(7)], device=DEV)
    assert codes.float().isnan().all(1).equal(bad) and scale.view(7, -1).isnan().all(1).equal(bad)
    assert scale.view(7, -1)[~bad].isfinite().all()
