"""Outputs of the prompt's calls whose parts would lie on one another are refused."""

import pytest
import torch

from carrykernel_b200 import _lib
from test_prompt_host import B, D, HV, N, lib, prefill, rotate  # noqa: F401


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


LIE_ON_ONE_ANOTHER = [
    torch.zeros(1, 4, D).expand(N, 4, D),
    torch.zeros(N, 1, D).expand(N, 4, D),
    torch.zeros(N * 4 * D).as_strided((N, 4, D), (D, D, 1)),
    torch.zeros(N * 4 * D).as_strided((N, 4, D), (4 * D - 2, D, 1)),
    torch.zeros(N * 4 * D).as_strided((N, 4, D), (D, N * D - 2, 1)),
]


@pytest.mark.parametrize("rows", LIE_ON_ONE_ANOTHER)
def test_heads_in_one_place(rows):
    for change in (dict(q=rows), dict(q_out=rows), dict(k=rows), dict(k=torch.zeros(N, 4, D), k_out=rows)):
        with pytest.raises(ValueError):
            rotate(**change)
    with pytest.raises(_lib.CudaUnavailable):             # what is only read may be one row for all
        rotate(q=rows, q_out=torch.zeros(N, 4, D))


@pytest.mark.parametrize("rows", [torch.zeros(4, N, D).transpose(0, 1), torch.zeros(N, 8, D + 2)[:, ::2, 1:-1], torch.zeros(N, 4, D)[::2].expand(3, 4, D)])
def test_heads_in_any_order_are_taken(rows):
    n = rows.shape[0]
    with pytest.raises(_lib.CudaUnavailable):
        rotate(q=rows, k=torch.zeros(n, 1, D)[:, :1].expand(n, 1, D), positions=torch.zeros(n, dtype=torch.int64))


def test_c_entry_refuses_heads_in_one_place(lib):  # noqa: F811
    a = _lib.RotateArgs()
    a.N, a.HQ, a.HK, a.D, a.axes = 5, 4, 4, D, 1
    a.q = a.k = a.q_out = a.k_out = a.q_weight = a.k_weight = a.positions = 4096        # looked at by no one: the call ends ahead of a launch
    for tok, head in ((0, D), (4 * D, 0), (D, D), (4 * D - 2, D), (D, 5 * D - 2), (-4 * D + 2, D)):
        for of in "qk":
            for name in "qk":
                bad = name == of
                setattr(a, f"stride_{name}_out_tok", tok if bad else 4 * D)
                setattr(a, f"stride_{name}_out_head", head if bad else D)
            assert lib.carry_gdn_qk_norm_rope(a, None) == -2
    a.HK = 0                                              # of no heads there is nothing that could
    a.stride_q_out_tok, a.stride_q_out_head, a.stride_k_out_tok, a.stride_k_out_head = 0, D, 0, 0
    assert lib.carry_gdn_qk_norm_rope(a, None) == -2
    a.HQ = a.HK = 0
    assert lib.carry_gdn_qk_norm_rope(a, None) == 0


@pytest.mark.gpu
def test_no_path_takes_them_on_a_gpu():
    """The native call path leaves them to the checks, and takes rows in any order."""
    from test_gpu_qk_norm_rope import BF16, DEV, check, make, qk_norm_rope
    q, k, start = torch.zeros(N, 4, D, device=DEV), torch.zeros(N, 2, D, device=DEV), torch.tensor([0, 3, N], dtype=torch.int32, device=DEV)
    call = dict(mixed_qkv=torch.zeros(N, 4 * D, device=DEV), a=torch.zeros(N, HV, device=DEV), b=torch.zeros(N, HV, device=DEV),
                A_log=torch.zeros(HV, device=DEV), dt_bias=torch.zeros(HV, device=DEV), out=torch.zeros(N, HV, D, device=DEV),
                final_state=torch.zeros(B, HV, D, D, device=DEV), query_start=start, max_query_len=3)
    prefill(**call)
    for change in (dict(final_state=call["final_state"][:1].expand(B, HV, D, D)), dict(out=call["out"][:1].expand(N, HV, D))):
        with pytest.raises(ValueError):
            prefill(**call | change)
    rest = [torch.ones(D, device=DEV), torch.ones(D, device=DEV), torch.zeros(10, D, device=DEV), torch.zeros(N, dtype=torch.int64, device=DEV)]
    qk_norm_rope(q, k, *rest)
    for rows in LIE_ON_ONE_ANOTHER:
        with pytest.raises(ValueError):
            qk_norm_rope(q, k, *rest, q_out=torch.zeros(2 * N * 4 * D, device=DEV).as_strided(rows.shape, rows.stride()))
    qkv, qw, kw, table, positions = make(N, 4, 2, D, D, BF16)
    out = torch.zeros(4, N, D, dtype=BF16, device=DEV).transpose(0, 1), torch.zeros(2, N, D, dtype=BF16, device=DEV).transpose(0, 1)
    qk_norm_rope(qkv[:, :4].to(DEV), qkv[:, 4:6].to(DEV), qw.to(DEV), kw.to(DEV), table.to(DEV), positions.to(DEV), q_out=out[0], k_out=out[1])
    check(out[0], qkv[:, :4], qw, table, positions)
    check(out[1], qkv[:, 4:6], kw, table, positions)
