"""Waits that run out in a call that is worked off in turns: the test-only twin of the library has smaller workspaces, and, of three value
heads, head 1's first copies never complete."""

import pytest
import torch

from carrykernel_b200 import _lib
from carrykernel_b200.vllm_integration import packed_prefill as pp
from test_gpu_prefill import BF16, DEV, F16, F32, make, run, starts
from test_gpu_wait_expiry import wait_test_library

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype,D,lengths", [(BF16, 64, [40001]), (F16, 128, [19000, 11000]), (F32, 64, [30000, 70, 1000]), (BF16, 128, [12000] * 4)], ids=str)
def test_later_turns_leave_the_head_as_it_was(dtype, D, lengths):
    """A request's later turns do not go on from a state that the first one never wrote; every other head has the numbers of a call in one turn."""
    HV = 3
    c, state = make(lengths, 1, HV, D, dtype, True)
    status = torch.zeros(1, dtype=torch.int32, device=DEV)
    want = run(c, state, lengths, HV, D, status=status)
    sizes = lambda: pp.prefill_workspace_bytes(c["mixed_qkv"].to(DEV), state.to(DEV), starts(lengths).to(DEV), max(lengths))  # noqa: E731
    whole = sizes()
    with wait_test_library():
        assert sizes() <= 2 ** 26 < whole
        out, final = run(c, state, lengths, HV, D, status=status)
    assert status.item() == _lib.STATUS_TIMEOUT
    assert out[:, 1].isnan().all() and final[:, 1].isnan().all()                     # what `run` fills its outputs with
    assert torch.equal(out[:, ::2], want[0][:, ::2]) and torch.equal(final[:, ::2], want[1][:, ::2])


@pytest.mark.parametrize("dtype", [BF16, F32])
def test_turns_of_late_warps(dtype):
    """No wait runs out: two and more turns have the numbers of one, twice over in the same workspace."""
    lengths, D, HV = [25000, 1, 3000], 64, 4
    c, state = make(lengths, 2, HV, D, dtype, True)
    status = torch.zeros(1, dtype=torch.int32, device=DEV)
    want = run(c, state, lengths, HV, D, status=status)
    with wait_test_library():
        work = torch.full((2 ** 26,), 255, dtype=torch.uint8, device=DEV)            # whatever it held
        for _ in range(2):
            out, final = run(c, state, lengths, HV, D, status=status, workspace=work)
            assert torch.equal(out, want[0]) and torch.equal(final, want[1])
    assert status.item() == 0
