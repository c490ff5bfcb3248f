"""Refusals of the prompt's calls (recurrence over sequences, norm and rotation), and their sizes, without a GPU."""

import ctypes as C
import os

import pytest
import torch

from carrykernel_b200 import _build, _lib
from carrykernel_b200.vllm_integration import packed_prefill as pp
from carrykernel_b200.vllm_integration.qk_norm_rope import qk_norm_rope
from oracle import prompt_oracle as orc

B, N, H, HV, D = 2, 6, 1, 2, 64


@pytest.fixture(scope="module", autouse=True)
def lib():
    if not os.path.exists(_lib.LIB_PATH):
        _build.build()
    return _lib.load_library()


def test_struct_sizes_match_header_layout():
    assert C.sizeof(_lib.PrefillArgs) == 18 * 8 + 14 * 4
    assert C.sizeof(_lib.RotateArgs) == 20 * 8 + 2 * 4 + 6 * 4 + 4 * 4 + 5 * 4 + 4


def prefill(**change):
    call = dict(mixed_qkv=torch.zeros(N, (2 * H + HV) * D), a=torch.zeros(N, HV), b=torch.zeros(N, HV), A_log=torch.zeros(HV),
                dt_bias=torch.zeros(HV), scale=1.0, out=torch.zeros(N, HV, D), final_state=torch.zeros(B, HV, D, D))
    call.update(change)
    return pp.gated_delta_rule_packed_prefill(**call)


def rotate(**change):
    call = dict(q=torch.zeros(N, 4, D), k=torch.zeros(N, 2, D), q_weight=torch.ones(D), k_weight=torch.ones(D), cos_sin=torch.zeros(10, D),
                positions=torch.zeros(N, dtype=torch.int64))
    call.update(change)
    return qk_norm_rope(**call)


def test_no_cpu_path():
    with pytest.raises(_lib.CudaUnavailable):
        prefill()
    with pytest.raises(_lib.CudaUnavailable):
        rotate()


START = torch.zeros(B + 1, dtype=torch.int32)


@pytest.mark.parametrize("change", [
    dict(mixed_qkv=torch.zeros(N, 1, (2 * H + HV) * D)),
    dict(mixed_qkv=torch.zeros(N, (2 * H + HV) * D - 1)),
    dict(mixed_qkv=torch.zeros(N, HV * D)),
    dict(mixed_qkv=torch.zeros(N, (2 * 4 + HV) * D)),                           # H = 4 does not divide HV = 2
    dict(mixed_qkv=torch.zeros((2 * H + HV) * D, N).T),
    dict(final_state=torch.zeros(HV, D, D)),
    dict(final_state=torch.zeros(B, HV, D, 2 * D)),
    dict(final_state=torch.zeros(B, HV, 32, 32)),
    dict(final_state=torch.zeros(B, HV, D, D, dtype=torch.bfloat16)),
    dict(final_state=torch.zeros(B, HV, D, D).transpose(2, 3)),
    dict(initial_state=torch.zeros(B + 1, HV, D, D)),
    dict(initial_state=torch.zeros(B, HV, D, D, dtype=torch.float64)),
    dict(initial_state=torch.zeros(B * HV * D * D + 1)[1:].view(B, HV, D, D)),
    dict(a=torch.zeros(N, HV + 1)),
    dict(b=torch.zeros(N - 1, HV)),
    dict(b=torch.zeros(N, HV, dtype=torch.bfloat16)),
    dict(a=torch.zeros(HV, N).T),
    dict(A_log=torch.zeros(HV + 1)),
    dict(dt_bias=torch.zeros(2 * HV)[::2]),
    dict(out=torch.zeros(N, HV, D + 1)),
    dict(out=torch.zeros(N, HV, 2 * D)[..., ::2]),
    dict(out=torch.zeros(N + 1, HV, D)),
    dict(max_query_len=N),                                                      # every request has N / B
    dict(final_state=torch.zeros(4, HV, D, D)),                                 # 6 rows for 4 requests
    dict(query_start=START),                                                    # no max_query_len
    dict(query_start=START, max_query_len=-1),
    dict(query_start=START.long(), max_query_len=3),
    dict(query_start=START[:-1], max_query_len=3),
    dict(status=torch.zeros(1)),
])
def test_prefill_refusals(change):
    with pytest.raises(ValueError):
        prefill(**change)


def test_prefill_refuses_unknown_types():
    with pytest.raises(TypeError):
        prefill(mixed_qkv=torch.zeros(N, (2 * H + HV) * D, dtype=torch.float64))
    with pytest.raises(TypeError):
        prefill(out=torch.zeros(N, HV, D, dtype=torch.int32))


@pytest.mark.parametrize("change", [
    dict(q=torch.zeros(N, 4 * D)),
    dict(k=torch.zeros(N + 1, 2, D)),
    dict(k=torch.zeros(N, 2, D, dtype=torch.bfloat16)),
    dict(q=torch.zeros(N, 4, 2 * D)[..., ::2]),
    dict(q=torch.zeros(N, 4, 63), k=torch.zeros(N, 2, 63)),
    dict(q=torch.zeros(N, 4, 514), k=torch.zeros(N, 2, 514), q_weight=torch.ones(514), k_weight=torch.ones(514)),
    dict(q_out=torch.zeros(N, 3, D)),
    dict(k_out=torch.zeros(N, 2, D, dtype=torch.float16)),
    dict(q_weight=torch.ones(D + 1)),
    dict(k_weight=torch.ones(D, dtype=torch.bfloat16)),
    dict(cos_sin=torch.zeros(10, D + 2)),
    dict(cos_sin=torch.zeros(10, 31)),
    dict(cos_sin=torch.zeros(D, 10).T),
    dict(cos_sin=torch.zeros(10)),
    dict(positions=torch.zeros(N)),
    dict(positions=torch.zeros(N - 1, dtype=torch.int64)),
    dict(positions=torch.zeros(3, N, dtype=torch.int64)),                       # no sections
    dict(positions=torch.zeros(3, N, dtype=torch.int64), sections=[16, 16]),
    dict(positions=torch.zeros(3, N, dtype=torch.int64), sections=[16, 16, 16]),
    dict(positions=torch.zeros(3, N, dtype=torch.int64), sections=[40, -16, 8]),
    dict(positions=torch.zeros(5, N, dtype=torch.int64), sections=[8, 8, 8, 4, 4]),
    dict(positions=torch.zeros(N, 3, dtype=torch.int64).T, sections=[16, 8, 8]),
    dict(eps=-1.0),
    dict(eps=float("nan")),
    dict(status=torch.zeros(2, dtype=torch.int32)),
])
def test_rotate_refusals(change):
    with pytest.raises(ValueError):
        rotate(**change)


def test_c_entries_refuse_what_they_cannot_index(lib):
    a = _lib.PrefillArgs()
    assert lib.carry_gdn_prefill(None, None) == -1 and lib.carry_gdn_prefill_workspace(None) == -1 and lib.carry_gdn_qk_norm_rope(None, None) == -1
    a.B, a.N, a.max_query, a.H, a.HV, a.K, a.V = 1, 100, 100, 1, 2, 64, 64
    assert lib.carry_gdn_prefill(a, None) == -1                                 # no pointers
    assert lib.carry_gdn_prefill_workspace(a) > 0
    for field, value, rc in (("B", -1, -2), ("max_query", 99, -2), ("H", 0, -2), ("HV", 65536, -8), ("K", 128, -5), ("qkv_dtype", 3, -3), ("N", -1, -2)):
        keep = getattr(a, field)
        setattr(a, field, value)
        assert lib.carry_gdn_prefill(a, None) == rc == lib.carry_gdn_prefill_workspace(a), field
        setattr(a, field, keep)
    a.N = a.max_query = 2 ** 30 + 1
    assert lib.carry_gdn_prefill(a, None) == -8 == lib.carry_gdn_prefill_workspace(a)
    a.N = a.max_query = 2 ** 30
    assert 0 < lib.carry_gdn_prefill_workspace(a) <= 1 << 30
    a.B = a.N = a.max_query = 0
    assert lib.carry_gdn_prefill(a, None) == 0 == lib.carry_gdn_prefill_workspace(a)
    r = _lib.RotateArgs()
    r.N, r.HQ, r.HK, r.D, r.rotary, r.axes = 3, 2, 1, 64, 64, 1
    r.sections[0] = 32
    assert lib.carry_gdn_qk_norm_rope(r, None) == -1
    for field, value, rc in (("N", -1, -2), ("D", 63, -2), ("D", 600, -5), ("rotary", 66, -2), ("axes", 0, -2), ("axes", 5, -2), ("eps", -1.0, -2),
                             ("dtype", 7, -3), ("table_dtype", -1, -3), ("HQ", 65536, -8), ("HK", 65536, -8)):
        keep = getattr(r, field)
        setattr(r, field, value)
        assert lib.carry_gdn_qk_norm_rope(r, None) == rc, field
        setattr(r, field, keep)
    r.N = 0
    assert lib.carry_gdn_qk_norm_rope(r, None) == 0


def test_workspace_sizes(lib):
    """Nothing for few tokens; within a bound, whatever the sizes; enough for every chunk where that is below it."""
    a = _lib.PrefillArgs()
    a.H, a.HV, a.K, a.V, a.qkv_dtype = 16, 32, 128, 128, _lib.BF16
    for B, T in ((1, 1), (64, 16), (3, 100), (1, 8192), (300, 500), (40000, 70), (1, 10 ** 7)):
        a.B, a.N, a.max_query = B, B * T, T
        need = lib.carry_gdn_prefill_workspace(a)
        assert 0 <= need <= 1 << 30 and (need > 0 or T <= 64)
    a.B, a.N, a.max_query = 0, 0, 0
    assert lib.carry_gdn_prefill_workspace(a) == 0


def test_oracle_recurrence_by_hand():
    """Two tokens of one head, by hand: write a value under a key, read it back, overwrite it in full."""
    D = 64
    q = torch.zeros(2, D)
    q[:, 3] = 2.0
    mixed = torch.cat([q, q, torch.arange(2 * D, dtype=torch.float32).view(2, D)], 1)
    out, state, _, _ = orc.delta_rule(mixed, torch.full((2, 1), -40.0), torch.full((2, 1), 40.0), torch.zeros(1), torch.zeros(1), 1.0, 1, D, [2])
    assert torch.allclose(out[:, 0], torch.arange(2 * D).view(2, D).double(), rtol=1e-6)
    assert torch.allclose(state[0, 0, :, 3], torch.arange(D, 2 * D).double(), rtol=1e-6) and state.abs().sum() - state[..., 3].abs().sum() < 1e-9


def test_oracle_rotation_by_hand():
    """A quarter turn takes a pair (y1, y2) to (-y2, y1)."""
    x = torch.arange(1.0, 9.0).view(1, 1, 8)
    cos_sin = torch.tensor([[1.0, 1.0, 0.0, 0.0], [0.0, 0.0, 1.0, 1.0]])
    y = x / (x ** 2).mean().sqrt()
    out, _ = orc.qk_norm_rope(x, torch.ones(8), cos_sin, torch.tensor([1]), 0.0)
    assert torch.allclose(out[0, 0].float(), (y * torch.tensor([0, 0, 1, 1, 1, 1, 1, 1.0])).view(8) + torch.cat([-y[0, 0, 2:4], y[0, 0, :2] - y[0, 0, 2:4], torch.zeros(4)]))
    out, _ = orc.qk_norm_rope(x, torch.ones(8), cos_sin, torch.tensor([[1], [0]]), 0.0, sections=[1, 1], interleaved=True)
    assert torch.allclose(out[0, 0, :4].float(), torch.stack([-y[0, 0, 1], y[0, 0, 0], y[0, 0, 2], y[0, 0, 3]]))
