"""Waits that run out ahead of the chains, in fp32: in the test-only twin of the library nothing announces the end of one of three products
for heads 1 to 3 of five, in the request's second chunk."""

import pytest
import torch

from carrykernel_b200 import _lib
from test_gpu_prefill import DEV, F32, goes_in_chunks, make, run
from test_gpu_wait_expiry import wait_test_library

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("D,H,lengths", [(64, 1, [200]), (128, 5, [150]), (64, 5, [200] * 20), (128, 1, [130] * 9)])
def test_a_chunk_that_was_not_worked_out_is_not_used(D, H, lengths):
    """Outputs of the chunk ahead of it are there; the head's further ones and its state are left as they were."""
    HV, n = 5, lengths[0]
    assert goes_in_chunks(lengths, F32)
    c, state = make(lengths, H, HV, D, F32, True)
    status = torch.zeros(1, dtype=torch.int32, device=DEV)
    want = run(c, state, lengths, HV, D, status=status)
    assert status.item() == 0
    with wait_test_library():
        out, final = run(c, state, lengths, HV, D, status=status)
    assert status.item() == _lib.STATUS_TIMEOUT
    rows = out.unflatten(0, (len(lengths), n))
    assert torch.equal(rows[:, :64], want[0].unflatten(0, (len(lengths), n))[:, :64])
    assert rows[:, 64:, 1:4].isnan().all() and final[:, 1:4].isnan().all()           # what `run` fills its outputs with
    assert torch.equal(out[:, ::4], want[0][:, ::4]) and torch.equal(final[:, ::4], want[1][:, ::4])
    status.zero_()
    again = run(c, state, lengths, HV, D, status=status)
    assert status.item() == 0 and torch.equal(again[0], want[0]) and torch.equal(again[1], want[1])


@pytest.mark.parametrize("D,B", [(64, 2), (128, 4)])
def test_outputs_ahead_of_the_chunk_are_all_there(D, B):
    """Whichever warp sees first that a chunk was not worked out, all have left what the chunk ahead of it gives."""
    HV, n = 5, 200
    c, state = make([n] * B, 1, HV, D, F32, True)
    want = run(c, state, [n] * B, HV, D)[0].unflatten(0, (B, n))
    with wait_test_library():
        for _ in range(30):
            out = run(c, state, [n] * B, HV, D)[0].unflatten(0, (B, n))
            assert torch.equal(out[:, :64], want[:, :64]) and out[:, 64:, 1:4].isnan().all()
