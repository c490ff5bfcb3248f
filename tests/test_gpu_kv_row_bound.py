"""The C entries of the key/value cache with a bound on a request's rows that is far beyond what there are: it says no more than the
number of rows does."""

import pytest
import torch

from oracle import hybrid_oracle as orc
from test_gpu_kv_cache import DEV, TYPES, check, make_cache, make_table, same

pytestmark = pytest.mark.gpu
MOST = 2 ** 31 - 1


def filled(tokens, dtype):
    g = torch.Generator().manual_seed(tokens)
    lengths, start = [tokens + 30, 90, tokens], [0, tokens, tokens + 1, 2 * tokens + 1]
    table, pages = make_table(lengths, 32, g)
    cache = make_cache(pages, 2, 32, 64, 16, g)
    rows = lambda heads: torch.randn(start[-1], heads, 64, generator=g).to(TYPES[dtype])  # noqa: E731
    return lengths, start, table, cache, rows


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("tokens", [1, 3, 50])
def test_attention(tokens, dtype):
    from carrykernel_b200 import _lib
    from carrykernel_b200.vllm_integration import quantized_kv_cache as qkv
    lib = _lib.load_library()
    lengths, start, table, cache, rows = filled(tokens, dtype)
    q = rows(4)
    on = [t.to(DEV) for t in (q, *cache, torch.full_like(q, 7.0), table, torch.tensor(lengths, dtype=torch.int32), torch.tensor(start, dtype=torch.int32))]
    args = qkv._attention_args(on[0], 0.125, *on[1:8], on[8], tokens, None)
    need = lib.carry_gdn_kv_attention_workspace(args)
    args.rows.max_query = q.shape[0]
    least = lib.carry_gdn_kv_attention_workspace(args)
    args.rows.max_query = MOST
    assert lib.carry_gdn_kv_attention_workspace(args) == least and need >= 0
    work = torch.empty(max(least, 16), dtype=torch.uint8, device=DEV)
    args.workspace, args.workspace_bytes = work.data_ptr(), work.numel()
    assert lib.carry_gdn_kv_attention(args, _lib.current_stream_ptr(on[0].device)) == 0
    torch.cuda.synchronize()
    check(on[5], q, 0.125, cache, table, lengths, dtype, query_start=start)


@pytest.mark.parametrize("tokens", [1, 50])
def test_append(tokens):
    from carrykernel_b200 import _lib
    from carrykernel_b200.vllm_integration import quantized_kv_cache as qkv
    lib = _lib.load_library()
    lengths, start, table, cache, rows = filled(tokens, "bf16")
    k, v = rows(2), rows(2)
    got = tuple(t.to(DEV) for t in cache)
    on = [t.to(DEV) for t in (k, v, table, torch.tensor(lengths, dtype=torch.int32), torch.tensor(start, dtype=torch.int32))]
    args = _lib.KvAppendArgs()
    qkv._rows(args.cache, args.rows, on[0], on[3], on[4], tokens, "k", on[0].device)
    qkv._cache(args.cache, *got, on[2], 3)
    args.k, args.stride_k_tok, args.stride_k_head = on[0].data_ptr(), on[0].stride(0), on[0].stride(1)
    args.v, args.stride_v_tok, args.stride_v_head = on[1].data_ptr(), on[1].stride(0), on[1].stride(1)
    args.dtype, args.rows.max_query = _lib.BF16, MOST
    assert lib.carry_gdn_kv_append(args, _lib.current_stream_ptr(on[0].device)) == 0
    torch.cuda.synchronize()
    same(tuple(t.cpu() for t in got), orc.append(k, v, cache, table, lengths, start))
