"""The 8-bit key/value cache on the GPU, append and attention, against their definitions in 64 bits.

Error bound of an output of the attention, with p the softmax weights: every weight is off by the error of its score
(fp32 sums: 2^-21 of the magnitudes behind it) and by its own rounding (2^-10 where queries are 16-bit, fp32 sums
included; 2^-18 where they are fp32), all of it relative to sum p |v|; then comes the rounding to out's type."""

import math
import os
import sys

import pytest
import torch

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))
from oracle import hybrid_oracle as orc  # noqa: E402

pytestmark = pytest.mark.gpu
DEV = "cuda"
TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
UNIT = {"bf16": 2.0 ** -8, "fp16": 2.0 ** -11, "fp32": 2.0 ** -23}
WEIGHT = {"bf16": 2.0 ** -10, "fp16": 2.0 ** -10, "fp32": 2.0 ** -18}


def make_table(lengths, page, g, extra=0, spare=2):
    """Pages in random order; the number of pages of the cache."""
    need = [-(-max(n, 0) // page) for n in lengths]
    order = (torch.randperm(sum(need) + spare, generator=g) + 1).tolist()
    table = torch.zeros(len(lengths), max(need, default=0) + extra, dtype=torch.int32)
    for b, n in enumerate(need):
        for i in range(n):
            table[b, i] = order.pop()
    return table, sum(need) + spare + 1


def make_cache(pages, HKV, page, D, block, g):
    out = []
    for _ in range(2):
        out.append((torch.randn(pages, HKV, page, D, generator=g) * 100).clamp(-448, 448).to(orc.F8))
        out.append(2.0 ** torch.randint(-9, -5, (pages, HKV, page // block), generator=g).float())
    return tuple(out)


def attend(q, scale, cache, table, lengths, query_start=None, max_query_len=None, out=None, **kw):
    from carrykernel_b200.vllm_integration import quantized_kv_cache as qkv
    cache = tuple(t.to(DEV) for t in cache)
    q = q if q.is_cuda else q.to(DEV)
    out = torch.full_like(q, 7.0) if out is None else out
    start = None if query_start is None else torch.tensor(query_start, dtype=torch.int32, device=DEV)
    got = qkv.quantized_paged_attention(q, scale, *cache, out, table.to(DEV),
                                        torch.tensor(lengths, dtype=torch.int32, device=DEV), query_start=start,
                                        max_query_len=max_query_len, **kw)
    torch.cuda.synchronize()
    return got


def check(got, q, scale, cache, table, lengths, dtype, query_start=None):
    out, weight, size = orc.attention(q.cpu(), scale, cache, table, lengths, query_start)
    bound = UNIT[dtype] * out.abs() + (WEIGHT[dtype] + 2.0 ** -21 * size) * weight + 1e-30
    off = (got.cpu().double() - out).abs()
    assert (off <= bound).all(), f"worst {(off / bound).max().item():.3g} of the bound"


def case(lengths, tokens, HQ, HKV, D, page, block, dtype, seed=0, query_start=None, extra=0, qscale=1.5):
    g = torch.Generator().manual_seed(seed)
    table, pages = make_table(lengths, page, g, extra)
    cache = make_cache(pages, HKV, page, D, block, g)
    N = len(lengths) * tokens if query_start is None else query_start[-1]
    q = (torch.randn(N, HQ, D, generator=g) * qscale).to(TYPES[dtype])
    got = attend(q, D ** -0.5, cache, table, lengths, query_start, tokens if query_start else None)
    check(got, q, D ** -0.5, cache, table, lengths, dtype, query_start)


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("D,page,block", [(64, 16, 16), (64, 128, 32), (128, 16, 16), (128, 48, 16), (128, 64, 64), (128, 256, 128)])
def test_one_token_a_request(D, page, block, dtype):
    case([1, 0, 15, 16, 17, 63, 64, 65, 130, 257], 1, 8, 2, D, page, block, dtype)


@pytest.mark.parametrize("HQ,HKV", [(1, 1), (3, 1), (16, 1), (20, 1), (6, 6), (40, 5)])
def test_head_groups(HQ, HKV):
    case([70, 33], 1, HQ, HKV, 128, 32, 32, "bf16")


@pytest.mark.parametrize("tokens", [2, 3, 5, 8, 17, 40, 70])
@pytest.mark.parametrize("dtype", ["bf16", "fp32"])
def test_several_tokens_a_request(tokens, dtype):
    """Some requests hold fewer tokens than they bring rows: rows at negative positions are zero."""
    case([tokens, tokens + 100, tokens - 1, 1, 0, 64 + tokens // 2], tokens, 4, 2, 64 if tokens % 2 else 128, 32, 16, dtype)


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("D", [64, 128])
def test_rows_of_every_number(dtype, D):
    case([5, 90, 33, 128, 200], 70, 4, 2, D, 64, 32, dtype, query_start=[0, 5, 5, 6, 76, 139])


def test_a_long_prompt_in_rows():
    case([300], 300, 2, 1, 128, 64, 32, "bf16")


@pytest.mark.parametrize("HQ,dtype", [(2, "bf16"), (8, "fp32")])
def test_a_long_context_is_split(HQ, dtype):
    case([20011, 3], 1, HQ, 1, 128, 128, 64, dtype, qscale=3.0)


def test_lengths_of_a_large_batch():
    g = torch.Generator().manual_seed(4)
    lengths = torch.randint(0, 200, (97,), generator=g).tolist()
    case(lengths, 1, 8, 4, 64, 32, 32, "fp16")


def test_table_wider_than_needed():
    case([40, 3], 1, 4, 2, 128, 16, 16, "bf16", extra=300)


def test_what_lies_beyond_a_length_is_not_read():
    """NaN codes and scales behind the last token, and in the pages of nobody."""
    g = torch.Generator().manual_seed(1)
    lengths, page, block = [1, 17, 50, 64, 100], 64, 16
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
    q = torch.randn(len(lengths) * 3, 4, 128, generator=g).bfloat16()
    got = attend(q, 0.1, cache, table, lengths)
    check(got, q, 0.1, clean, table, lengths, "bf16")


@pytest.mark.parametrize("tokens", [4, 80])
def test_a_nan_key_reaches_only_the_rows_that_see_it(tokens):
    g = torch.Generator().manual_seed(2)
    lengths, page = [tokens + 9], 32
    table, pages = make_table(lengths, page, g)
    cache = make_cache(pages, 1, page, 64, 32, g)
    q = torch.randn(tokens, 2, 64, generator=g).bfloat16()
    at = lengths[0] - 2                                  # the second last token: two rows see it
    cache[0].view(torch.uint8)[int(table[0][at // page]), 0, at % page, 3] = 0x7f
    got = attend(q, 0.125, cache, table, lengths)
    assert got[-2:].isnan().all() and got[:-2].isfinite().all()


def test_infinite_and_nan_queries_stay_in_their_rows():
    g = torch.Generator().manual_seed(3)
    lengths = [50, 50]
    table, pages = make_table(lengths, 32, g)
    cache = make_cache(pages, 2, 32, 64, 32, g)
    q = torch.randn(8, 4, 64, generator=g)
    bad = q.clone()
    bad[1, 2, 5], bad[6, 0, 63] = math.nan, math.inf
    for dt in TYPES.values():
        good, got = attend(q.to(dt), 0.125, cache, table, lengths), attend(bad.to(dt), 0.125, cache, table, lengths)
        hit = torch.zeros(8, 4, dtype=torch.bool, device=DEV)
        hit[1, 2] = hit[6, 0] = True
        assert got.isnan().any(-1).equal(hit) and torch.equal(got[~hit], good[~hit])


@pytest.mark.parametrize("kscale,vscale,qmul", [(2.0 ** -100, 2.0 ** 100, 1.0), (2.0 ** 60, 2.0 ** -60, 2.0 ** -60), (1.0, 1.0, 2.0 ** -100), (2.0 ** -8, 2.0 ** -30, 300.0)])
def test_scales_of_every_size(kscale, vscale, qmul):
    """Neither codes nor weights leave the range of the type that the products are formed in."""
    g = torch.Generator().manual_seed(6)
    lengths = [100, 31]
    table, pages = make_table(lengths, 32, g)
    cache = list(make_cache(pages, 2, 32, 128, 16, g))
    cache[1], cache[3] = torch.full_like(cache[1], kscale), cache[3] * vscale
    q = (torch.randn(2, 4, 128, generator=g) * qmul).bfloat16()
    scale = 0.05 / (100 * kscale * qmul) if qmul < 100 else 0.1
    got = attend(q, scale, cache, table, lengths)
    check(got, q, scale, cache, table, lengths, "bf16")


def test_value_blocks_of_very_different_scales():
    """The block with the largest values has hardly any weight: the others' values still come out in full."""
    g = torch.Generator().manual_seed(8)
    lengths = [96]
    table, pages = make_table(lengths, 32, g)
    cache = make_cache(pages, 1, 32, 64, 16, g)
    q = torch.randn(1, 2, 64, generator=g).bfloat16()
    cache[3].fill_(2.0 ** -12)
    last = int(table[0][2])
    cache[3][last, 0, 1] = 2.0 ** 6
    cache[2][last, 0, 16:] = 0
    got = attend(q, 0.125, cache, table, lengths)
    check(got, q, 0.125, cache, table, lengths, "bf16")


def test_strides_of_q_out_and_pages():
    from carrykernel_b200.vllm_integration import quantized_kv_cache as qkv
    g = torch.Generator().manual_seed(7)
    lengths = [33, 70, 5]
    table, pages = make_table(lengths, 16, g)
    cache = make_cache(pages, 2, 16, 64, 16, g)
    both = torch.zeros(pages, 2, 2, 16, 64, dtype=orc.F8, device=DEV)      # keys and values of a page side by side
    both[:, 0], both[:, 1] = cache[0].to(DEV), cache[2].to(DEV)
    for shift in (0, 1):
        wide = torch.randn(3, 4 * 64 + 100, generator=g).bfloat16().to(DEV)
        q = wide[:, shift:shift + 256].view(3, 4, 64)
        frame = torch.full((4, 3, 80), 5.0, dtype=torch.bfloat16, device=DEV)
        out = frame[:, :, shift:shift + 64].transpose(0, 1)                # heads in front
        qkv.quantized_paged_attention(q, 0.125, both[:, 0], cache[1].to(DEV), both[:, 1], cache[3].to(DEV), out,
                                      torch.cat([table, table], 1).to(DEV)[:, :table.shape[1]],
                                      torch.tensor(lengths, dtype=torch.int32, device=DEV))
        check(out, q, 0.125, cache, table, lengths, "bf16")
        assert (frame[:, :, :shift] == 5).all() and (frame[:, :, shift + 64:] == 5).all()


def test_padding_pages_and_bad_ids_are_skipped_and_flagged():
    g = torch.Generator().manual_seed(10)
    lengths, page = [100, 100, 100, 10 ** 6], 32
    table, pages = make_table([100, 100, 100, 128], page, g)
    table[0, 1], table[1, 0] = 0, -3
    cache = make_cache(pages, 2, page, 64, 32, g)
    q = torch.randn(4, 4, 64, generator=g).half()
    status = torch.zeros(1, dtype=torch.int32, device=DEV)
    good = lengths[:3] + [128]
    check(attend(q, 0.125, cache, table, good, status=status), q, 0.125, cache, table, good, "fp16")
    assert status.item() == 0
    table[2, 2] = pages + 5
    check(attend(q, 0.125, cache, table, lengths, status=status), q, 0.125, cache, table, lengths, "fp16")
    assert status.item() == 4


def test_query_ranges_outside_of_the_call_are_skipped_and_flagged():
    g = torch.Generator().manual_seed(11)
    lengths = [40, 50]
    table, pages = make_table(lengths, 32, g)
    cache = make_cache(pages, 1, 32, 64, 32, g)
    q = torch.randn(6, 2, 64, generator=g).bfloat16()
    status = torch.zeros(1, dtype=torch.int32, device=DEV)
    got = attend(q, 0.125, cache, table, lengths, query_start=[0, 3, 900], max_query_len=3, status=status)
    check(got, q, 0.125, cache, table, lengths, "bf16", query_start=[0, 3, 900])
    assert status.item() == 4


def test_the_same_call_twice_gives_the_same_bits_on_any_stream_and_in_a_graph():
    from carrykernel_b200.vllm_integration import quantized_kv_cache as qkv
    g = torch.Generator().manual_seed(12)
    for lengths, tokens in (([3000, 1, 700], 1), ([130, 200, 80], 80)):
        table, pages = make_table(lengths, 64, g)
        cache = tuple(t.to(DEV) for t in make_cache(pages, 2, 64, 128, 32, g))
        q = torch.randn(3 * tokens, 8, 128, generator=g).bfloat16().to(DEV)
        want = attend(q, 0.1, cache, table, lengths).clone()
        table, lens = table.to(DEV), torch.tensor(lengths, dtype=torch.int32, device=DEV)
        out = torch.zeros_like(want)
        need = qkv.attention_workspace_bytes(q, cache[0], cache[1], table)
        work = torch.full((need + 16,), 255, dtype=torch.uint8, device=DEV)
        stream = torch.cuda.Stream()
        stream.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(stream):
            qkv.quantized_paged_attention(q, 0.1, *cache, out, table, lens, workspace=work)
        stream.synchronize()
        assert torch.equal(out, want)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            qkv.quantized_paged_attention(q, 0.1, *cache, out, table, lens)
        for _ in range(2):
            out.zero_()
            graph.replay()
            torch.cuda.synchronize()
            assert torch.equal(out, want)


# ---- append ------------------------------------------------------------------------------------------------------------------

def append(k, v, cache, table, lengths, query_start=None, max_query_len=None, status=None):
    from carrykernel_b200.vllm_integration import quantized_kv_cache as qkv
    got = tuple(t.to(DEV) for t in cache)
    start = None if query_start is None else torch.tensor(query_start, dtype=torch.int32, device=DEV)
    k, v = (t if t.is_cuda else t.to(DEV) for t in (k, v))
    qkv.quantized_kv_append(k, v, *got, table.to(DEV), torch.tensor(lengths, dtype=torch.int32, device=DEV),
                            query_start=start, max_query_len=max_query_len, status=status)
    torch.cuda.synchronize()
    return tuple(t.cpu() for t in got)


def same(a, b):
    for x, y in zip(a, b):
        assert torch.equal(x.view(torch.uint8) if x.dtype == orc.F8 else x, y.view(torch.uint8) if y.dtype == orc.F8 else y)


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("D,page,block", [(64, 16, 16), (128, 64, 32), (128, 128, 128), (64, 96, 48)])
@pytest.mark.parametrize("lengths,tokens,start", [
    ([1, 17, 16, 40, 2, 0], 1, None), ([5, 130, 3, 200, 37], 5, None), ([7, 300, 256, 9], 150, [0, 7, 157, 157, 164])])
def test_append(D, page, block, dtype, lengths, tokens, start):
    """Bit for bit: every step of it is exact, or rounded once.  Requests with fewer tokens than rows among them."""
    g = torch.Generator().manual_seed(D + page + tokens)
    table, pages = make_table(lengths, page, g, extra=1)
    cache = make_cache(pages, 2, page, D, block, g)
    N = start[-1] if start else tokens * len(lengths)
    k, v = (torch.randn(N, 2, D, generator=g) * torch.exp(2 * torch.randn(N, 2, 1, generator=g)) * s for s in (3.0, 1.0))
    k, v = k.to(TYPES[dtype]), v.to(TYPES[dtype])
    same(append(k, v, cache, table, lengths, start, tokens if start else None), orc.append(k, v, cache, table, lengths, start))


def test_a_block_filled_token_by_token_has_the_codes_of_one_filled_at_once():
    g = torch.Generator().manual_seed(20)
    table = torch.tensor([[2, 1]], dtype=torch.int32)
    cache = make_cache(3, 2, 32, 64, 32, g)
    k, v = (torch.randn(50, 2, 64, generator=g) * 2.0 ** torch.randint(-2, 4, (50, 2, 1), generator=g) for _ in range(2))
    once = append(k, v, cache, table, [50])
    step = cache
    for n in range(50):
        step = append(k[n:n + 1], v[n:n + 1], step, table, [n + 1])
    assert torch.equal(once[1][1:], step[1][1:]) and torch.equal(once[3][1:], step[3][1:])
    for a, b in ((once[0], step[0]), (once[2], step[2])):
        a, b = a.float(), b.float()
        normal = (a.abs() >= 2.0 ** -6) & (b.abs() >= 2.0 ** -6)
        assert torch.equal(a[normal], b[normal]) and ((a - b).abs() <= 2.0 ** -9).all()


def test_numbers_that_are_not_finite_mark_their_token_and_no_other():
    g = torch.Generator().manual_seed(21)
    table, cache = torch.tensor([[1]], dtype=torch.int32), make_cache(2, 2, 32, 64, 32, g)
    k, v = (torch.randn(20, 2, 64, generator=g) for _ in range(2))
    k[3, 0, 1], k[8, 1, 0], v[12, 0, 63], v[19, 1, 7] = math.nan, math.inf, -math.inf, math.nan
    got = append(k, v, cache, table, [20])
    same(got, orc.append(k, v, cache, table, [20]))
    assert got[2].float()[1, :, :20].isfinite().all() and (got[1][1] < 1).all()


@pytest.mark.parametrize("size", [0.0, 1e-38, 2.0 ** -110, 448.0, 448.1, 3e38])
def test_append_of_zeros_and_of_extreme_numbers(size):
    g = torch.Generator().manual_seed(22)
    table, cache = torch.tensor([[1]], dtype=torch.int32), make_cache(2, 1, 16, 64, 16, g)
    k = torch.full((16, 1, 64), size) * torch.sign(torch.randn(16, 1, 64, generator=g))
    same(append(k, k, cache, table, [16]), orc.append(k, k, cache, table, [16]))


def test_append_skips_padding_and_flags_what_lies_outside():
    g = torch.Generator().manual_seed(23)
    table = torch.tensor([[1, 0], [3, 9], [-1, 2]], dtype=torch.int32)
    cache = make_cache(4, 2, 16, 64, 16, g)
    k, v = (torch.randn(60, 2, 64, generator=g).bfloat16() for _ in range(2))
    status = torch.zeros(1, dtype=torch.int32, device=DEV)
    same(append(k, v, cache, table, [20, 20, 30], status=status), orc.append(k, v, cache, table, [20, 20, 30]))
    assert status.item() == 4


def test_append_strides_and_alignment():
    g = torch.Generator().manual_seed(24)
    table, cache = torch.tensor([[1, 2]], dtype=torch.int32), make_cache(3, 2, 16, 64, 16, g)
    for shift in (0, 3):
        wide = torch.randn(20, 300, generator=g).half().to(DEV)
        k = wide[:, shift:shift + 128].view(20, 2, 64)
        v = torch.randn(2, 20, 64, generator=g).half().to(DEV).transpose(0, 1)
        same(append(k, v, cache, table, [20]), orc.append(k.cpu(), v.cpu(), cache, table, [20]))


def behind_a_padding_page(t):
    raw = t.view(torch.uint8) if t.dtype == orc.F8 else t
    return torch.cat([torch.zeros_like(raw[:1]), raw]).view(t.dtype)


def test_pages_beyond_two_to_the_31_bytes():
    """A page whose codes start past 2^31: written, and read back by the attention."""
    page, D, HKV = 128, 128, 8
    pages = 2 ** 31 // (page * D * HKV) + 3
    from carrykernel_b200.vllm_integration import quantized_kv_cache as qkv
    cache = qkv.init_quantized_kv(pages, HKV, page, D, DEV, block=64)
    g = torch.Generator().manual_seed(25)
    table, lens = torch.tensor([[pages - 1, pages - 2]], dtype=torch.int32), torch.tensor([200], dtype=torch.int32, device=DEV)
    k, v = (torch.randn(200, HKV, D, generator=g).bfloat16() for _ in range(2))
    qkv.quantized_kv_append(k.to(DEV), v.to(DEV), *cache, table.to(DEV), lens)
    q = torch.randn(1, HKV, D, generator=g).bfloat16()
    out = qkv.quantized_paged_attention(q.to(DEV), 0.1, *cache, torch.zeros_like(q, device=DEV), table.to(DEV), lens)
    small, near = tuple(behind_a_padding_page(t[-2:].cpu()) for t in cache), torch.tensor([[2, 1]], dtype=torch.int32)
    empty = qkv.init_quantized_kv(3, HKV, page, D, "cpu", block=64)
    same(small, orc.append(k, v, empty, near, [200]))
    check(out, q, 0.1, small, near, [200], "bf16")
