"""Attention and append with row ranges at the ends of 32 bits: nothing outside of the call's rows is read or written, and what has
rows is done."""

import pytest
import torch

from test_gpu_kv_cache import DEV, TYPES, make_cache, make_table

pytestmark = pytest.mark.gpu
LEAST, MOST = -2 ** 31, 2 ** 31 - 1


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("tokens", [3, 50])
def test_row_ranges_at_the_ends_of_32_bits(tokens, dtype):
    from carrykernel_b200 import _lib
    from carrykernel_b200.vllm_integration import quantized_kv_cache as qkv
    g = torch.Generator().manual_seed(tokens)
    lengths = [tokens + 30, 90]
    table, pages = make_table(lengths, 32, g)
    cache = [t.to(DEV) for t in make_cache(pages, 2, 32, 64, 16, g)]
    table, lengths = table.to(DEV), torch.tensor(lengths, dtype=torch.int32, device=DEV)
    q, k, v = (torch.randn(tokens + 9, heads, 64, generator=g).to(TYPES[dtype]).to(DEV) for heads in (4, 2, 2))

    def calls(start):
        start = torch.tensor(start, dtype=torch.int32, device=DEV)
        status, guarded = torch.zeros(1, dtype=torch.int32, device=DEV), torch.full((tokens + 9 + 64, 4, 64), 9.0, dtype=q.dtype, device=DEV)
        qkv.quantized_paged_attention(q, 0.125, *cache, guarded[32:32 + tokens + 9], table, lengths, start, tokens, status=status)
        filled = [t.clone() for t in cache]
        qkv.quantized_kv_append(k, v, *filled, table, lengths, start, tokens, status=status)
        return guarded, filled, status.item()

    want, want_cache, clean = calls([0, tokens, tokens])
    assert clean == 0
    for start in ([0, tokens, LEAST], [0, tokens, LEAST + tokens]):
        got, got_cache, status = calls(start)
        assert status == _lib.STATUS_BAD_RANGE, start
        assert torch.equal(got, want) and (got[32 + tokens:] == 9).all()
        assert all(torch.equal(x.view(torch.uint8), y.view(torch.uint8)) for x, y in zip(got_cache, want_cache)), start
