"""The norms of keys in the gated delta rule over whole sequences: the state behind a token that forgets all ahead of it is one product."""

import pytest
import torch

from test_gpu_prefill import BF16, F16, F32, goes_in_chunks, make, run

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("D", [64, 128])
def test_a_token_that_forgets_leaves_beta_v_k(dtype, D):
    """With a last decay of exp(-200) the state is beta v k^T / |k|.

    The sum of squares: D / 16 products on the tensor cores, each cut at 2^-23 of the sum so far, and a step for all that is smaller; half of
    that for its root, 4.5 * 2^-23.  The sigmoid, two multiplications, and the sum that forms the state: 2^-23 each at most.  Less than 2^-20."""
    B, H, HV, n = 8, 2, 4, 127
    c, state = make([n] * B, H, HV, D, dtype, True, gates=F32)
    c["A_log"], c["dt_bias"] = torch.zeros(HV), torch.zeros(HV)
    last = torch.arange(1, B + 1) * n - 1
    c["a"][last] = 200.0                                  # softplus of it is 200
    assert goes_in_chunks([n], dtype)
    _, final = run(c, state, [n] * B, HV, D)
    x = c["mixed_qkv"][last].double()
    k, v = x[:, H * D:2 * H * D].view(B, H, D).repeat_interleave(HV // H, 1), x[:, 2 * H * D:].view(B, HV, D)
    k = k / torch.sqrt((k * k).sum(-1, keepdim=True) + 1e-6)
    want = torch.sigmoid(c["b"][last].double())[..., None, None] * v[..., None] * k[:, :, None]
    off = (final.cpu().double() - want).flatten(2).norm(dim=-1) / want.flatten(2).norm(dim=-1)
    assert (off <= 2.0 ** -20).all(), f"{off.max():.2e}"
