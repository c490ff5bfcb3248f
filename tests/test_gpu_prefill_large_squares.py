"""The gated delta rule over whole sequences with the norm, where squares pass fp32: NaN, and no zeros in its place."""

import pytest
import torch

from test_gpu_prefill import BF16, F32, make, run

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("n,at", [(30, 7), (130, 7), (200, 64), (200, 199)])
def test_queries_and_keys_whose_squares_pass_fp32(dtype, D, n, at):
    H, HV = 2, 4
    c, state = make([n], H, HV, D, dtype, True)
    clean = run(c, state, [n], HV, D)
    query = dict(c, mixed_qkv=c["mixed_qkv"].clone())
    query["mixed_qkv"][at, D:2 * D] = 1e20
    out, final = run(query, state, [n], HV, D)
    spoilt = torch.zeros_like(out, dtype=torch.bool)
    spoilt[at, 2:] = True                                 # the heads that read it
    assert out[spoilt].isnan().all() and torch.equal(out[~spoilt], clean[0][~spoilt]) and torch.equal(final, clean[1])
    key = dict(c, mixed_qkv=c["mixed_qkv"].clone())
    key["mixed_qkv"][at, H * D + D:H * D + 2 * D] = 1e20
    out, final = run(key, state, [n], HV, D)
    assert out[at:, 2:].isnan().all() and final[:, 2:].isnan().all()
    ahead = at if dtype == BF16 or n <= 96 else at // 64 * 64
    assert torch.equal(out[:ahead], clean[0][:ahead]) and torch.equal(out[:, :2], clean[0][:, :2]) and torch.equal(final[:, :2], clean[1][:, :2])
