"""Keys that nobody norms, in the gated delta rule over whole sequences: finite ones of any size are keys like others."""

import pytest
import torch

from oracle import prompt_oracle as orc
from test_gpu_prefill import BF16, F16, F32, check, goes_in_chunks, make, run

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("n,at", [(30, 7), (130, 7), (130, 64), (200, 199)])
def test_a_key_whose_squares_pass_fp32_and_that_writes_nothing(dtype, D, n, at):
    """beta = sigmoid(-200), which is 0 in fp32: the token decays the state and no more."""
    H, HV = 2, 4
    c, state = make([n], H, HV, D, dtype, True, l2norm=False, gates=F32)
    c["mixed_qkv"][at, H * D + D:H * D + 2 * D] = 1e20
    c["b"][at] = -200.0
    got = run(c, state, [n], HV, D, l2norm=False)
    assert got[0].isfinite().all() and got[1].isfinite().all()
    c["mixed_qkv"][at, H * D + D:H * D + 2 * D] = 0.0
    check(got, c, state, [n], H, D, l2norm=False, in_chunks=goes_in_chunks([n], dtype), rows=[i for i in range(n) if i != at])


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("n", [30, 130])
def test_a_key_whose_squares_pass_fp32_and_that_is_written(dtype, n):
    """The first token writes v k^T with |k| above 1.8e19 into a state of zeros; later keys are of length 1, and what they take of it is as large.

    T's entries are good to 2^-18, and fewer than 32 of a token's chunk weigh in full (beta below 1, keys of no one direction): 2^-13 of the state."""
    H, HV, D = 1, 2, 64
    c, _ = make([n], H, HV, D, dtype, l2norm=False, gates=F32)
    c["mixed_qkv"][0, D:2 * D] = torch.linspace(2e18, 6e18, D).to(dtype)
    c["A_log"], c["dt_bias"], c["a"] = torch.zeros(HV), torch.full((HV,), -4.0), torch.zeros(n, HV)
    assert c["mixed_qkv"][0, D:2 * D].float().square().sum() == float("inf")
    _, final = run(c, None, [n], HV, D, l2norm=False)
    want = orc.delta_rule(**{k: v for k, v in c.items() if k != "mixed_qkv"}, mixed=c["mixed_qkv"], H=H, D=D, lengths=[n], l2norm=False)[1]
    assert want.norm() > 1e17
    assert (final.cpu().double() - want).norm() <= 2.0 ** -13 * want.norm()


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("bad", [float("inf"), float("-inf"), float("nan")])
def test_a_key_that_is_not_finite_among_large_ones(dtype, D, bad):
    """Every place of a row: the state is spoilt from that token on, and no token ahead of it is."""
    H, HV, n = 1, 1, 100
    c, state = make([n], H, HV, D, dtype, True, l2norm=False, gates=F32)
    if dtype == BF16:
        c["mixed_qkv"][40, D:2 * D] = 1e20
        c["b"][40] = -200.0
    clean = run(c, state, [n], HV, D, l2norm=False)
    for column in range(0, D, 7):
        d = dict(c, mixed_qkv=c["mixed_qkv"].clone())
        at = 41 + column % 59
        d["mixed_qkv"][at, D + column] = bad
        out, final = run(d, state, [n], HV, D, l2norm=False)
        assert torch.equal(out[:at], clean[0][:at]) and not out[at:].isfinite().any() and not final.isfinite().any()
