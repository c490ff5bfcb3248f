"""The 8-bit key/value attention over numbers of requests: clusters of one to eight CTAs to a (request, head), and prompts
whose last CTAs, those that do not fill the GPU, are cut along the context.  Oracle and error bound are those of
test_gpu_kv_cache."""

import pytest
import torch

from test_gpu_kv_cache import TYPES, attend, case, check, make_cache, make_table

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("requests,context", [(5, 1000), (40, 600), (70, 500), (100, 300), (200, 100), (250, 500), (300, 100)])
@pytest.mark.parametrize("dtype,D,tokens", [("bf16", 128, 1), ("fp32", 64, 1), ("fp16", 64, 5), ("fp32", 128, 5)])
def test_numbers_of_requests(requests, context, dtype, D, tokens):
    lengths = [max((context * (37 * b % 101)) // 100, tokens) for b in range(requests - 1)] + [context]
    case(lengths, tokens, 2, 1, D, 32, 16, dtype, seed=requests)


@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
def test_many_requests_cut_along_the_context(dtype):
    """160 CTAs, one to a request, and contexts that are worth the cut: long ones, short ones and one that ends in the first part."""
    lengths = [4096, 1500, 1030, 17, 0] + [20 + b % 60 for b in range(155)]
    case(lengths, 17, 1, 1, 64, 64, 32, dtype, seed=8)


@pytest.mark.parametrize("length,tokens", [(4600, 2600), (4600, 2561), (8000, 2400)])
def test_the_first_rows_of_a_prompt_are_cut(length, tokens):
    """16 heads of ten or eleven tiles of 256 rows: the last tiles are whole, the first are cut."""
    g = torch.Generator().manual_seed(tokens)
    table, pages = make_table([length], 64, g)
    cache = make_cache(pages, 16, 64, 64, 32, g)
    q = torch.randn(tokens, 16, 64, generator=g).to(TYPES["bf16"])
    out = attend(q, 0.125, cache, table, [length]).cpu()
    for first in (0, 127, 253, 511, 767, 1279, tokens - 3):
        rows = slice(first, first + 3)
        check(out[rows], q[rows], 0.125, cache, table, [length - tokens + first + 3], "bf16")


@pytest.mark.parametrize("dtype", ["bf16", "fp32"])
@pytest.mark.parametrize("rows", [1, 20])
def test_rows_of_no_request(rows, dtype):
    """Rows that no request claims are left as they are."""
    g = torch.Generator().manual_seed(9)
    cache = make_cache(3, 2, 32, 64, 32, g)
    q = torch.randn(rows, 4, 64, generator=g).to(TYPES[dtype])
    table = torch.zeros(0, 4, dtype=torch.int32)
    out = attend(q, 0.125, cache, table, [], query_start=[0], max_query_len=rows)
    assert (out == 7).all()
