"""The 8-bit key/value attention where one way of working ends and the next begins: short and long contexts, few and many
rows, contexts cut into parts.  Oracle and error bound are those of test_gpu_kv_cache."""

import math

import pytest
import torch

from oracle import hybrid_oracle as orc
from test_gpu_kv_cache import DEV, TYPES, attend, case, check, make_cache, make_table

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("context", [2047, 4095, 4096, 4097, 8193])
@pytest.mark.parametrize("dtype", ["bf16", "fp32"])
def test_context_lengths_about_the_end_of_the_cluster_kernel(context, dtype):
    case([context, 5], 1, 2, 1, 128, 64, 32, dtype, seed=context)
    case([context], 2, 2, 1, 64, 32, 32, dtype, seed=context)


@pytest.mark.parametrize("rows", [7, 8, 9, 15, 16, 17, 33])
def test_numbers_of_rows_about_the_tiles(rows):
    for dtype in TYPES:
        case([300, 20], rows, 1, 1, 128 if rows % 2 else 64, 64, 16, dtype, seed=rows)


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("D,lengths,tokens", [(128, [1500, 40, 1100], 20), (64, [2100], 40)])
def test_contexts_cut_into_parts(D, lengths, tokens, dtype):
    """Few (request, head)s, many rows: the context is cut; one request ends inside the first part."""
    case(lengths, tokens, 2, 1, D, 64, 32, dtype, seed=tokens)


def test_rows_of_every_number_over_parts():
    case([1300, 1290, 10, 0], 45, 2, 2, 128, 128, 64, "bf16", query_start=[0, 45, 46, 56, 60])


@pytest.mark.parametrize("tokens", [1, 20])
@pytest.mark.parametrize("context", [200, 1500])
def test_scores_and_values_that_keep_growing(tokens, context):
    """Every block outdoes the one before, in its keys and, elsewhere, in its values: maxima and units are replaced again
    and again, by small and by large steps."""
    g = torch.Generator().manual_seed(1)
    table, pages = make_table([context], 16, g)
    cache = list(make_cache(pages, 1, 16, 128, 16, g))
    for j, page in enumerate(table[0].tolist()):
        cache[1][page] = 2.0 ** (-9 + 6 * j / (context / 16))
        cache[3][page] = 2.0 ** ((5 * j) % 23 - 12)
    q = torch.randn(tokens, 8, 128, generator=g).bfloat16()
    got = attend(q, 128 ** -0.5, cache, table, [context])
    check(got, q, 128 ** -0.5, cache, table, [context], "bf16")


@pytest.mark.parametrize("dtype", ["bf16", "fp32"])
def test_many_rows_read_nothing_beyond_a_length(dtype):
    g = torch.Generator().manual_seed(2)
    lengths, page, block = [40, 50, 64, 100, 1100], 64, 16
    table, pages = make_table(lengths, page, g, extra=2)
    cache = make_cache(pages, 2, page, 128, block, g)
    clean = tuple(t.clone() for t in cache)
    mine = torch.zeros(pages, page, dtype=torch.bool)
    for b, n in enumerate(lengths):
        for j in range(n):
            mine[int(table[b][j // page]), j % page] = True
    for codes, scale in (cache[:2], cache[2:]):
        codes.view(torch.uint8).permute(0, 2, 1, 3)[~mine] = 0x7f
        scale.permute(0, 2, 1)[~mine.view(pages, -1, block).any(2)] = math.nan
    q = torch.randn(len(lengths) * 30, 4, 128, generator=g).to(TYPES[dtype])
    check(attend(q, 0.1, cache, table, lengths), q, 0.1, clean, table, lengths, dtype)


@pytest.mark.parametrize("dtype", ["fp16", "fp32"])
def test_many_rows_skip_padding_pages(dtype):
    g = torch.Generator().manual_seed(3)
    lengths = [200, 150]
    table, pages = make_table(lengths, 32, g)
    table[0, 2], table[1, 0] = 0, pages + 7
    cache = make_cache(pages, 1, 32, 64, 32, g)
    q = torch.randn(60, 2, 64, generator=g).to(TYPES[dtype])
    status = torch.zeros(1, dtype=torch.int32, device=DEV)
    check(attend(q, 0.125, cache, table, lengths, status=status), q, 0.125, cache, table, lengths, dtype)
    assert status.item() == 4


def test_many_rows_with_strides():
    from carrykernel_b200.vllm_integration import quantized_kv_cache as qkv
    g = torch.Generator().manual_seed(4)
    lengths = [90, 40]
    table, pages = make_table(lengths, 16, g)
    cache = make_cache(pages, 2, 16, 64, 16, g)
    for shift in (0, 1):
        wide = torch.randn(80, 4 * 64 + 100, generator=g).bfloat16().to(DEV)
        q = wide[:, shift:shift + 256].view(80, 4, 64)
        frame = torch.full((4, 80, 80), 5.0, dtype=torch.bfloat16, device=DEV)
        out = frame[:, :, shift:shift + 64].transpose(0, 1)
        qkv.quantized_paged_attention(q, 0.125, *(t.to(DEV) for t in cache), out, table.to(DEV),
                                      torch.tensor(lengths, dtype=torch.int32, device=DEV))
        check(out, q, 0.125, cache, table, lengths, "bf16")
        assert (frame[:, :, :shift] == 5).all() and (frame[:, :, shift + 64:] == 5).all()


def test_negative_scale():
    for tokens in (1, 40):
        g = torch.Generator().manual_seed(5)
        table, pages = make_table([130], 64, g)
        cache = make_cache(pages, 1, 64, 64, 32, g)
        q = torch.randn(tokens, 2, 64, generator=g).bfloat16()
        check(attend(q, -0.2, cache, table, [130]), q, -0.2, cache, table, [130], "bf16")


@pytest.mark.parametrize("lengths,tokens", [([5000, 12], 1), ([900], 1), ([1400], 30)])
def test_a_call_repeated_gives_the_same_bits(lengths, tokens):
    g = torch.Generator().manual_seed(6)
    table, pages = make_table(lengths, 64, g)
    cache = tuple(t.to(DEV) for t in make_cache(pages, 1, 64, 128, 64, g))
    q = torch.randn(len(lengths) * tokens, 4, 128, generator=g).bfloat16().to(DEV)
    want = attend(q, 0.1, cache, table, lengths).clone()
    for _ in range(5):
        assert torch.equal(attend(q, 0.1, cache, table, lengths), want)
