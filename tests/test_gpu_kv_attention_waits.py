"""The waits of the many-row attention over the 8-bit key/value cache, in the test-only twin of the library, where every
softmax warp comes microseconds late to a quarter of its steps."""

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
