"""The waits of the many-row attention over the 8-bit key/value cache, in the test-only twin of the library, where every
softmax warp comes microseconds late to a quarter of its steps, and, in caches of three heads, the first copies of request 0's
head 1 never complete."""

import pytest
import torch

from test_gpu_kv_cache import DEV, TYPES, attend, check, make_cache, make_table
from test_gpu_wait_expiry import wait_test_library

pytestmark = pytest.mark.gpu


def made(lengths, tokens, HQ, HKV, D, dtype, seed):
    g = torch.Generator().manual_seed(seed)
    table, pages = make_table(lengths, 64, g)
    cache = make_cache(pages, HKV, 64, D, 32, g)
    q = torch.randn(len(lengths) * tokens, HQ, D, generator=g).to(TYPES[dtype])
    return q, D ** -0.5, cache, table, lengths


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("lengths,tokens,HQ,HKV", [([1000, 70, 700], 64, 2, 1), ([900, 333], 150, 4, 2), ([2600], 40, 1, 1)])
def test_a_late_warp_misses_no_phase(lengths, tokens, HQ, HKV, D):
    """One row tile and two, contexts whole and cut into parts.  A warp that comes to a step when the copies and conversions
    of the next three are done finds its own all the same."""
    call = made(lengths, tokens, HQ, HKV, D, "bf16", seed=D + tokens)
    status = torch.zeros(1, dtype=torch.int32, device=DEV)
    want = attend(*call, status=status)
    with wait_test_library():
        got = attend(*call, status=status)
    assert status.item() == 0 and torch.equal(got, want)
    check(got, *call, "bf16")


@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("lengths,tokens", [([130, 200], 80), ([1500, 1300, 20], 40), ([3000], 300)])
def test_rows_of_a_wait_that_runs_out_are_left_as_they_were(lengths, tokens, dtype):
    """Contexts whole and cut into parts: the other rows come out as they should, nothing is joined from what is missing."""
    from carrykernel_b200 import _lib
    call = made(lengths, tokens, 6, 3, 128, dtype, seed=tokens)
    status = torch.zeros(1, dtype=torch.int32, device=DEV)
    want = attend(*call, status=status)
    assert status.item() == 0
    with wait_test_library():
        got = attend(*call, status=status)
    assert status.item() == _lib.STATUS_TIMEOUT
    want[:tokens, 2:4] = 7.0                             # what `attend` fills its output with
    assert torch.equal(got, want)
    status.zero_()
    want = attend(*call, status=status)
    assert status.item() == 0
    check(want, *call, dtype)


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("lengths,tokens,HQ,HKV", [([4000, 900], 300, 2, 2), ([1300] * 40, 40, 8, 4), ([130, 64, 65, 700], 260, 1, 1)])
def test_warps_of_every_kind_that_come_late(lengths, tokens, HQ, HKV, D):
    """Those that fetch, convert and issue as well: long rows of steps, several CTAs to an SM's turn, value scales that move the
    rows' units, contexts that end inside a step."""
    q, scale, cache, table, lengths = made(lengths, tokens, HQ, HKV, D, "fp16", seed=tokens)
    g = torch.Generator().manual_seed(D)
    cache[3].copy_(2.0 ** torch.randint(-20, -4, cache[3].shape, generator=g).float())
    status = torch.zeros(1, dtype=torch.int32, device=DEV)
    want = attend(q, scale, cache, table, lengths, status=status)
    with wait_test_library():
        got = attend(q, scale, cache, table, lengths, status=status)
    assert status.item() == 0 and torch.equal(got, want)
