"""Append to blocks that already hold tokens under a scale of some other make: no power of two, or beyond those that append
writes itself.  A value is code * scale whatever the scale; oracle and comparison, bit for bit, are those of test_gpu_kv_cache."""

import pytest
import torch

from oracle import hybrid_oracle as orc
from test_gpu_kv_cache import TYPES, append, make_cache, make_table, same

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("D,page,block", [(64, 32, 16), (128, 64, 64), (128, 128, 128)])
@pytest.mark.parametrize("tokens", [1, 7, 40])
def test_blocks_under_scales_of_another_make(tokens, D, page, block, dtype):
    """Scales that stay, that grow to a power of two, and, among whole numbers, quotients that are halfway between two codes."""
    g = torch.Generator().manual_seed(D + block + tokens)
    lengths = [tokens + n for n in (5, 11, 20, 33, 63, 90, 100)]
    table, pages = make_table(lengths, page, g)
    cache = list(make_cache(pages, 2, page, D, block, g))
    for i in (1, 3):
        cache[i] = torch.rand(cache[i].shape, generator=g) * 2.0 ** torch.randint(-9, 2, cache[i].shape, generator=g)
    cache[1][::2] = 0.75                                 # whole numbers times this over it
    k, v = (torch.randn(len(lengths) * tokens, 2, D, generator=g) * s for s in (1.0, 3.0))
    k = torch.where(torch.rand(k.shape, generator=g) < 0.5, torch.randint(-300, 301, k.shape, generator=g) * 0.75, k)
    k, v = k.to(TYPES[dtype]), v.to(TYPES[dtype])
    same(append(k, v, cache, table, lengths), orc.append(k, v, cache, table, lengths))


@pytest.mark.parametrize("old", [0.0, 2.0 ** -140, 3e-39, 2.0 ** 126, 2.0 ** 127, 1.5 * 2.0 ** 126, 3e38])
def test_scales_at_the_ends_of_fp32(old):
    g = torch.Generator().manual_seed(7)
    table, cache = torch.tensor([[1]], dtype=torch.int32), list(make_cache(2, 1, 32, 64, 32, g))
    cache[1].fill_(old), cache[3].fill_(old)
    k = torch.randn(4, 1, 64, generator=g) * (old * 100 if 1 < old < 1e37 else 1e38 if old > 1 else 1.0)
    same(append(k, k, cache, table, [20]), orc.append(k, k, cache, table, [20]))
