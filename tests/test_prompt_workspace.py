"""The size of a prompt's workspace goes by sizes alone: nothing is read or allocated for it."""

import pytest
import torch

from carrykernel_b200.vllm_integration import packed_prefill as pp
from test_prompt_host import lib  # noqa: F401


class NothingAllocated(torch.overrides.TorchFunctionMode):
    def __torch_function__(self, func, types, args=(), kwargs=None):
        assert func not in (torch.empty, torch.zeros, torch.ones, torch.empty_like, torch.full, torch.tensor), func
        return func(*args, **(kwargs or {}))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_workspace_of_tensors_without_memory(dtype):
    """As many bytes for rows of one token's memory, for states of one request's and for neither, as for whole ones."""
    B, T, H, HV, D = 3, 200, 2, 4, 64
    width = (2 * H + HV) * D
    whole = torch.zeros(B * T, width, dtype=dtype), torch.zeros(B, HV, D, D)
    need = pp.prefill_workspace_bytes(*whole)
    assert need > 0
    for device in ("cpu", "meta"):
        mixed, state = torch.zeros(1, width, dtype=dtype, device=device), torch.zeros(1, HV, D, D, device=device)
        with NothingAllocated():
            assert pp.prefill_workspace_bytes(mixed.expand(B * T, width), state.expand(B, HV, D, D)) == need
    start = torch.zeros(B + 1, dtype=torch.int32)
    with NothingAllocated():
        assert pp.prefill_workspace_bytes(*whole, start, T) > 0 and pp.prefill_workspace_bytes(*whole, start, 3) == 0


def test_sizes_that_are_no_call_are_refused():
    mixed, state = torch.zeros(6, 4 * 64), torch.zeros(2, 2, 64, 64)
    for change in (dict(mixed_qkv=mixed[None]), dict(mixed_qkv=mixed[:, 1:]), dict(mixed_qkv=mixed[:5]), dict(final_state=state[0]),
                   dict(final_state=torch.zeros(2, 2, 64, 32)), dict(max_query_len=4), dict(query_start=torch.zeros(3, dtype=torch.int32))):
        with pytest.raises(ValueError):
            pp.prefill_workspace_bytes(**{"mixed_qkv": mixed, "final_state": state, **change})
    with pytest.raises(TypeError):
        pp.prefill_workspace_bytes(mixed.double(), state)
