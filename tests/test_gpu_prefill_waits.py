"""The waits of the gated delta rule in chunks, in the test-only twin of the library, where warps of every kind come microseconds late to
some of their chunks, and, of three value heads, the first copies of head 1's first chunk never complete."""

import pytest
import torch

from carrykernel_b200 import _lib
from test_gpu_prefill import BF16, DEV, F16, F32, goes_in_chunks, make, run
from test_gpu_wait_expiry import wait_test_library

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("D,H,HV,lengths", [(64, 2, 4, [700]), (128, 1, 2, [300, 130]), (128, 8, 16, [520, 1, 64, 300]), (64, 16, 32, [130] * 6)])
def test_a_late_warp_misses_no_phase(D, H, HV, lengths, dtype):
    """One CTA to a processor and two, tiles of one stage and of two, requests that end inside a chunk: the same numbers."""
    assert goes_in_chunks(lengths, dtype)
    c, state = make(lengths, H, HV, D, dtype, True)
    status = torch.zeros(1, dtype=torch.int32, device=DEV)
    want = run(c, state, lengths, HV, D, status=status)
    with wait_test_library():
        got = run(c, state, lengths, HV, D, status=status)
    assert status.item() == 0 and torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("D,B", [(64, 1), (128, 2), (128, 20)])
def test_a_head_whose_wait_runs_out_is_left_as_it_was(D, B, dtype):
    lengths = [200] * B
    c, state = make(lengths, 1, 3, D, dtype, True)
    status = torch.zeros(1, dtype=torch.int32, device=DEV)
    want = run(c, state, lengths, 3, D, status=status)
    assert status.item() == 0
    with wait_test_library():
        got = run(c, state, lengths, 3, D, status=status)
    assert status.item() == _lib.STATUS_TIMEOUT
    for x, y in zip(got, want):
        assert x[:, 1].isnan().all()                     # what `run` fills its outputs with
        assert torch.equal(x[:, ::2], y[:, ::2])
    status.zero_()
    again = run(c, state, lengths, 3, D, status=status)
    assert status.item() == 0 and torch.equal(again[0], want[0]) and torch.equal(again[1], want[1])
