"""The gated delta rule over whole sequences from states, and with gates, that are not finite."""

import pytest
import torch

from test_gpu_prefill import BF16, F16, F32, check, goes_in_chunks, make, run

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("n", [1, 30, 130])
@pytest.mark.parametrize("bad", [float("inf"), float("-inf"), float("nan")])
def test_a_number_of_the_initial_state_spoils_its_row_and_no_other(dtype, D, n, bad):
    H, HV, lengths = 1, 2, [n, n]
    c, state = make(lengths, H, HV, D, dtype, True)
    clean = run(c, state, lengths, HV, D)
    state[1, 1, 5, D - 3] = bad
    out, final = run(c, state, lengths, HV, D)
    rows, rows_state = torch.zeros_like(out, dtype=torch.bool), torch.zeros_like(final, dtype=torch.bool)
    rows[n:, 1, 5], rows_state[1, 1, 5] = True, True
    assert not out[rows].isfinite().any() and not final[rows_state].isfinite().any()
    if goes_in_chunks(lengths, dtype):
        assert out[rows].isnan().all() and final[rows_state].isnan().all()
    assert torch.equal(out[~rows], clean[0][~rows]) and torch.equal(final[~rows_state], clean[1][~rows_state])


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("n", [30, 130])
def test_infinite_inputs_of_gates_are_gates_of_0_and_1(dtype, n):
    """A decay input of infinity forgets all, one of minus infinity nothing; a write strength's input writes all or nothing."""
    H, HV, D = 1, 4, 64
    c, state = make([n], H, HV, D, dtype, True, gates=F32)
    c["A_log"] = torch.zeros(HV)
    ends = torch.tensor([float("inf"), float("-inf")]).repeat(n)[:n]
    c["a"][3::7, 0], c["a"][5:40:3, 1] = float("inf"), float("-inf")
    c["b"][:, 2], c["b"][:, 3] = ends, ends.roll(1)
    got = run(c, state, [n], HV, D)
    limits = dict(c, a=c["a"].clamp(-300, 300), b=c["b"].clamp(-300, 300))          # exp(-300) is 0 in fp32
    assert got[0].isfinite().all() and got[1].isfinite().all()
    check(got, limits, state, [n], H, D, in_chunks=goes_in_chunks([n], dtype))
