"""Residual addition and norm where a block of threads takes row after row: more rows than the GPU has room for at once, of
widths on and off the 16-byte grid, for each way that a row is spread over lanes."""

import pytest
import torch

pytestmark = pytest.mark.gpu

from test_gpu_residual_norm import DEV, call, check  # noqa: E402

BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32


@pytest.mark.parametrize("grouped", [False, True])
@pytest.mark.parametrize("types", [(BF16, BF16), (F32, F32), (BF16, F32), (F16, BF16)])
@pytest.mark.parametrize("N,W", [(9999, 100), (9500, 256), (9000, 255), (5500, 400), (5000, 511), (3000, 1024), (2500, 2050), (1300, 4096),
                                 (1400, 4095), (700, 8191), (620, 9001), (610, 12288), (310, 20001)])
def test_many_rows(N, W, types, grouped):
    g = torch.Generator().manual_seed(N + W)
    x, r = (torch.randn(N, W, generator=g).to(t).to(DEV) for t in types)
    w = (1 + 0.1 * torch.randn(W, generator=g)).to(types[0]).to(DEV)
    before, want = r.clone(), (x.float() + r.float()).to(types[1])
    check(x, before, w, grouped, *call(x, r, w, grouped))
    assert torch.equal(r, want)
