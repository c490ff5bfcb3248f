"""The 8-bit key/value attention where the value scales of a context's blocks lie far apart, over the whole range that append
writes (2^-100 for a block of zeros, up to 2^119).  Oracle and error bound are those of test_gpu_kv_cache: an output is off by
2^-10 of its own sum p |v|, whatever other rows see and however large a block is that it hardly weighs.  fp16 weights keep that
bound: they are full down to 2^-21 of the largest weight times scale, and what is below is 2^-32 of it at most."""

import pytest
import torch

from test_gpu_kv_cache import TYPES, attend, check, make_cache, make_table

pytestmark = pytest.mark.gpu


def made(context, tokens, D, dtype, seed, HQ=2):
    g = torch.Generator().manual_seed(seed)
    table, pages = make_table([context], 64, g)
    cache = list(make_cache(pages, 1, 64, D, 16, g))
    q = torch.randn(tokens, HQ, D, generator=g).to(TYPES[dtype])
    return q, cache, table, g


def block_of(table, n):
    """Page and place in it of the context's n-th block of 16 tokens."""
    return int(table[0][n // 4]), n % 4


def run(q, cache, table, context, dtype):
    scale = q.shape[2] ** -0.5
    got = attend(q, scale, cache, table, [context])
    check(got, q, scale, cache, table, [context], dtype)


def zeros_beside(power, tokens, D, dtype):
    """Blocks of zeros, as append writes them, beside blocks of a large scale."""
    q, cache, table, _ = made(180, tokens, D, dtype, power)
    cache[3].fill_(2.0 ** power)
    for n in (0, 3, 5, 6, 11):
        page, at = block_of(table, n)
        cache[3][page, 0, at] = 2.0 ** -100
        cache[2][page, 0, at * 16:at * 16 + 16] = 0
    run(q, cache, table, 180, dtype)


def unseen(power, tokens, D, dtype):
    """A block of large values that most rows come before, in the step that they end in."""
    q, cache, table, _ = made(128, tokens, D, dtype, power)
    cache[3].fill_(2.0 ** -9)
    page, at = block_of(table, 7)
    cache[3][page, 0, at] = 2.0 ** (power - 9)
    run(q, cache, table, 128, dtype)


def hardly_weighed(power, tokens, D, dtype):
    """Half of the blocks have values 2^power times the others' and weights of about 2^-power times theirs, or less."""
    q, cache, table, _ = made(300, tokens, D, dtype, power)
    cache[3].fill_(2.0 ** -9)
    cache[0].view(torch.uint8)[..., 0] = 0x70            # 128: column 0 of a key decides, against the others' some 2^-3 each
    cache[1].fill_(2.0 ** -11)
    q[..., 0] = power * 0.693 * 16 * D ** 0.5
    for n in range(0, 19, 2):
        page, at = block_of(table, n)
        cache[3][page, 0, at] = 2.0 ** (power - 9)
        cache[0].view(torch.uint8)[page, 0, at * 16:at * 16 + 16, 0] = 0
    run(q, cache, table, 300, dtype)


def of_every_size(seed, tokens, D, dtype, context=700):
    q, cache, table, g = made(context, tokens, D, dtype, seed)
    cache[3].copy_(2.0 ** torch.randint(-100, 110, cache[3].shape, generator=g).float())
    run(q, cache, table, context, dtype)


MANY = [(20, 128, "bf16"), (150, 64, "bf16")]


@pytest.mark.parametrize("tokens,D,dtype", MANY)
@pytest.mark.parametrize("power", [15, 21, 28, 34, 36, 60, 119])
def test_many_rows_blocks_of_zeros_beside_large_values(power, tokens, D, dtype):
    zeros_beside(power, tokens, D, dtype)


@pytest.mark.parametrize("tokens,D,dtype", MANY[:1] + [(100, 64, "bf16")])
@pytest.mark.parametrize("power", [20, 26, 33, 50, 100])
def test_many_rows_large_values_that_a_row_does_not_see(power, tokens, D, dtype):
    unseen(power, tokens, D, dtype)


@pytest.mark.parametrize("tokens,D,dtype", MANY)
@pytest.mark.parametrize("power", [10, 24, 40, 90])
def test_many_rows_large_values_of_little_weight(power, tokens, D, dtype):
    hardly_weighed(power, tokens, D, dtype)


@pytest.mark.parametrize("tokens,D,dtype", MANY + [(400, 128, "bf16")])
@pytest.mark.parametrize("seed", range(3))
def test_many_rows_scales_of_every_size(seed, tokens, D, dtype):
    of_every_size(seed, tokens, D, dtype)


# few rows, by clusters (short contexts) and by the line, and many fp32 rows
FEW = [(1, 128, "bf16"), (4, 64, "bf16"), (8, 128, "bf16"), (4, 128, "fp32"), (8, 64, "fp32"), (40, 128, "fp32"), (70, 64, "fp32")]


@pytest.mark.parametrize("tokens,D,dtype", FEW)
@pytest.mark.parametrize("power", [21, 36, 100])
def test_few_rows_blocks_of_zeros_beside_large_values(power, tokens, D, dtype):
    zeros_beside(power, tokens, D, dtype)


@pytest.mark.parametrize("tokens,D,dtype", FEW[1:])
@pytest.mark.parametrize("power", [26, 33, 50, 100])
def test_few_rows_large_values_that_a_row_does_not_see(power, tokens, D, dtype):
    unseen(power, tokens, D, dtype)


@pytest.mark.parametrize("tokens,D,dtype", FEW)
@pytest.mark.parametrize("power", [10, 24, 40, 90])
def test_few_rows_large_values_of_little_weight(power, tokens, D, dtype):
    hardly_weighed(power, tokens, D, dtype)


@pytest.mark.parametrize("tokens,D,dtype", FEW)
@pytest.mark.parametrize("seed", range(3))
def test_few_rows_scales_of_every_size(seed, tokens, D, dtype):
    of_every_size(seed, tokens, D, dtype)
    of_every_size(seed, tokens, D, dtype, context=9000)


@pytest.mark.parametrize("dtype", ["bf16", "fp32"])
@pytest.mark.parametrize("context,tokens", [(60, 1), (180, 8), (1500, 1), (9000, 2), (9000, 8), (60, 40), (9000, 40)])
def test_values_at_the_end_of_the_range(context, tokens, dtype):
    """448 * 2^119 throughout, which is what comes out: no sum on the way leaves fp32.  Contexts in one piece, in a cluster's, in
    CTAs' and in parts."""
    q, cache, table, _ = made(context, tokens, 128, dtype, tokens)
    cache[2].fill_(448.0)
    cache[3].fill_(2.0 ** 119)
    run(q, cache, table, context, dtype)


@pytest.mark.parametrize("zero", [2.0 ** -100, 0.0])
@pytest.mark.parametrize("power", [15, 24, 40])
@pytest.mark.parametrize("context,first", [(300, 1), (700, 8), (3000, 64)])
@pytest.mark.parametrize("tokens,D,dtype", FEW + MANY)
def test_blocks_of_zeros_that_have_nearly_all_the_weight(tokens, D, dtype, context, first, power, zero):
    """The `first` blocks and then every fourth have scores that are `power` above the others' in log2, and values that are all
    zero: the others' small weights are all that comes out."""
    q, cache, table, _ = made(context, tokens, D, dtype, power)
    cache[3].fill_(2.0 ** -9)
    cache[0].view(torch.uint8)[..., 0] = 0
    cache[1].fill_(2.0 ** -11)
    q[..., 0] = power * 0.693 * 16 * D ** 0.5
    for n in range((context + 15) // 16):
        if n < first or n % 4 == 0:
            page, at = block_of(table, n)
            rows = slice(at * 16, at * 16 + 16)
            cache[3][page, 0, at], cache[2][page, 0, rows] = zero, 0
            cache[0].view(torch.uint8)[page, 0, rows, 0] = 0x70
    run(q, cache, table, context, dtype)
