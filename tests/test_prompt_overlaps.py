"""Outputs of the prompt's calls whose parts would lie on one another are refused, without a GPU."""

import pytest
import torch

from carrykernel_b200 import _lib
from test_prompt_host import B, D, HV, N, lib, prefill  # noqa: F401


@pytest.mark.parametrize("state", [
    torch.zeros(1, HV, D, D).expand(B, HV, D, D),
    torch.zeros((HV + 1) * D * D).as_strided((B, HV, D, D), (D * D, D * D, D, 1)),
])
def test_states_of_two_requests_in_one_place(state):
    with pytest.raises(ValueError):
        prefill(final_state=state)
    with pytest.raises(_lib.CudaUnavailable):
        prefill(initial_state=state)                      # a state to begin with may be one for all
    with pytest.raises(_lib.CudaUnavailable):
        prefill(final_state=state[:1])


def test_c_entry_refuses_states_of_two_requests_in_one_place(lib):  # noqa: F811
    a = _lib.PrefillArgs()
    a.B, a.N, a.max_query, a.H, a.HV, a.K, a.V = 2, 6, 3, 1, HV, D, D
    a.final_state = a.A_log = a.dt_bias = a.mixed_qkv = a.a = a.b = a.out = 4096        # looked at by no one: the call ends ahead of a launch
    a.stride_out_tok = HV * D
    for stride in (0, HV * D * D - 4, -4):
        a.stride_final_req = stride
        assert lib.carry_gdn_prefill(a, None) == -2


@pytest.mark.parametrize("out", [
    torch.zeros(1, HV, D).expand(N, HV, D),
    torch.zeros(N * HV * D).as_strided((N, HV, D), (D, D, 1)),
])
def test_outputs_of_two_tokens_in_one_place(out):
    with pytest.raises(ValueError):
        prefill(out=out)


def test_c_entry_refuses_outputs_of_two_tokens_in_one_place(lib):  # noqa: F811
    a = _lib.PrefillArgs()
    a.B, a.N, a.max_query, a.H, a.HV, a.K, a.V = 1, 6, 6, 1, HV, D, D
    a.final_state = a.A_log = a.dt_bias = a.mixed_qkv = a.a = a.b = a.out = 4096
    for stride in (0, HV * D - 1, -1):
        a.stride_out_tok = stride
        assert lib.carry_gdn_prefill(a, None) == -2
