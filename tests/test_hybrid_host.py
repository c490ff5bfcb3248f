"""Refusals of the key/value cache's and the layer norm's calls, and their sizes, without a GPU."""

import ctypes as C
import os

import pytest
import torch

from carrykernel_b200 import _build, _lib
from carrykernel_b200.vllm_integration import quantized_kv_cache as qkv
from carrykernel_b200.vllm_integration.residual_norm import add_rms_norm_quant
from oracle import hybrid_oracle as orc


@pytest.fixture(scope="module", autouse=True)
def lib():
    if not os.path.exists(_lib.LIB_PATH):
        _build.build()
    return _lib.load_library()


def test_struct_sizes_match_header_layout():
    assert C.sizeof(_lib.KvCache) == 4 * 8 + 4 * 8 + 3 * 8 + 6 * 4
    assert C.sizeof(_lib.KvRows) == 8 + 3 * 4 + 4
    assert C.sizeof(_lib.KvAppendArgs) == C.sizeof(_lib.KvCache) + C.sizeof(_lib.KvRows) + 6 * 8 + 8 + 8
    assert C.sizeof(_lib.KvAttentionArgs) == C.sizeof(_lib.KvCache) + C.sizeof(_lib.KvRows) + 8 * 8 + 4 * 4 + 8
    assert C.sizeof(_lib.NormArgs) == 6 * 8 + 4 * 8 + 7 * 4 + 4


def test_init_and_bytes():
    kc, ks, vc, vs = qkv.init_quantized_kv(5, 2, 64, 128, "cpu", block=16)
    assert kc.shape == vc.shape == (5, 2, 64, 128) and ks.shape == vs.shape == (5, 2, 4)
    assert qkv.kv_bytes_per_token(2, 128, 16) == 2 * 2 * 128 + 2 * 2 * 4 / 16
    for page, D, block in ((60, 128, 15), (64, 96, 32), (64, 128, 48), (0, 128, 16), (256, 128, 256)):
        with pytest.raises(ValueError):
            qkv.init_quantized_kv(5, 2, page, D, "cpu", block=block)


def call(**change):
    cache = qkv.init_quantized_kv(5, 2, 64, 128, "cpu", block=32)
    a = dict(q=torch.zeros(3, 4, 128), scale=1.0, k_codes=cache[0], k_scale=cache[1], v_codes=cache[2], v_scale=cache[3],
             out=torch.zeros(3, 4, 128), block_table=torch.zeros(3, 2, dtype=torch.int32),
             lengths=torch.ones(3, dtype=torch.int32))
    a.update(change)
    return qkv.quantized_paged_attention(**a)


def test_no_cpu_path():
    with pytest.raises(_lib.CudaUnavailable):
        call()
    with pytest.raises(_lib.CudaUnavailable):
        append()
    with pytest.raises(_lib.CudaUnavailable):
        norm()


BAD_CACHE = [
    dict(k_codes=torch.zeros(5, 2, 64, 128, dtype=torch.int8)),
    dict(v_codes=torch.zeros(5, 2, 64, 64).to(qkv.CODES)),
    dict(k_codes=torch.zeros(5, 2, 64, 256).to(qkv.CODES)[..., :128]),
    dict(k_scale=torch.zeros(5, 2, 3)),
    dict(k_scale=torch.zeros(5, 2, 8)),
    dict(v_scale=torch.zeros(5, 2, 4)),
    dict(v_scale=torch.zeros(5, 2, 2, dtype=torch.float64)),
    dict(block_table=torch.zeros(2, 2, dtype=torch.int32)),
    dict(block_table=torch.zeros(3, 2, dtype=torch.int64)),
    dict(lengths=torch.ones(3, dtype=torch.int64)),
    dict(lengths=torch.ones(3, 1, dtype=torch.int32)),
    dict(query_start=torch.zeros(4, dtype=torch.int32)),                        # no max_query_len
    dict(query_start=torch.zeros(3, dtype=torch.int32), max_query_len=1),
    dict(query_start=torch.zeros(4, dtype=torch.int64), max_query_len=1),
    dict(max_query_len=2),
    dict(status=torch.zeros(1)),
]


@pytest.mark.parametrize("change", BAD_CACHE + [
    dict(q=torch.zeros(3, 3, 128), out=torch.zeros(3, 3, 128)),
    dict(q=torch.zeros(4, 4, 128), out=torch.zeros(4, 4, 128)),
    dict(q=torch.zeros(3, 4, 64)),
    dict(q=torch.zeros(3, 128, 4).transpose(1, 2)),
    dict(out=torch.zeros(3, 4, 64)),
    dict(out=torch.zeros(3, 4, 128).half()),
], ids=lambda c: "-".join(c))
def test_attention_refuses(change):
    with pytest.raises(ValueError):
        call(**change)


def test_attention_refuses_other_types():
    with pytest.raises(TypeError):
        call(q=torch.zeros(3, 4, 128).double(), out=torch.zeros(3, 4, 128).double())


def append(**change):
    cache = qkv.init_quantized_kv(5, 2, 64, 128, "cpu", block=32)
    a = dict(k=torch.zeros(3, 2, 128), v=torch.zeros(3, 2, 128), k_codes=cache[0], k_scale=cache[1], v_codes=cache[2],
             v_scale=cache[3], block_table=torch.zeros(3, 2, dtype=torch.int32), lengths=torch.ones(3, dtype=torch.int32))
    a.update(change)
    return qkv.quantized_kv_append(**a)


@pytest.mark.parametrize("change", BAD_CACHE + [
    dict(k=torch.zeros(3, 4, 128)),
    dict(v=torch.zeros(3, 2, 64)),
    dict(v=torch.zeros(3, 2, 128).half()),
    dict(v=torch.zeros(3, 128, 2).transpose(1, 2)),
], ids=lambda c: "-".join(c))
def test_append_refuses(change):
    with pytest.raises(ValueError):
        append(**change)


def norm(**change):
    a = dict(x=torch.zeros(4, 300), residual=torch.zeros(4, 300), weight=torch.zeros(300),
             codes=torch.zeros(4, 300).to(torch.float8_e4m3fn), scale=torch.zeros(4))
    a.update(change)
    return add_rms_norm_quant(**a)


@pytest.mark.parametrize("change", [
    dict(x=torch.zeros(4, 2, 150)),
    dict(x=torch.zeros(300, 4).T),
    dict(residual=torch.zeros(4, 301)),
    dict(residual_out=torch.zeros(4, 300).half()),
    dict(weight=torch.zeros(299)),
    dict(weight=torch.zeros(600)[::2]),
    dict(codes=torch.zeros(4, 300)),
    dict(scale=torch.zeros(4, 2)),
    dict(scale=torch.zeros(4, dtype=torch.float16)),
    dict(x=torch.zeros(1, 40000), residual=None, weight=torch.zeros(40000), codes=torch.zeros(1, 40000).to(qkv.CODES), scale=torch.zeros(1)),
], ids=lambda c: "-".join(c))
def test_norm_refuses(change):
    with pytest.raises(ValueError):
        norm(**change)


def test_library_refuses_bad_arguments_itself(lib):
    a = _lib.KvAttentionArgs()
    assert lib.carry_gdn_kv_attention(None, None) == -1 and lib.carry_gdn_kv_append(None, None) == -1
    assert lib.carry_gdn_add_rms_norm_quant(None, None) == -1 and lib.carry_gdn_kv_attention_workspace(None) == -1
    assert lib.carry_gdn_kv_attention(a, None) == -2
    c = a.cache
    c.HKV, c.page, c.block, c.D, c.num_pages, c.max_pages = 2, 64, 32, 128, 4, 2
    a.rows.B, a.rows.N, a.rows.max_query, a.HQ = 2, 2, 1, 4
    a.dtype = 7
    assert lib.carry_gdn_kv_attention(a, None) == -3
    a.dtype = 1
    assert lib.carry_gdn_kv_attention(a, None) == -1                            # no q
    c.D = 96
    assert lib.carry_gdn_kv_attention(a, None) == _lib.ERR_UNSUPPORTED
    c.D, a.HQ = 128, 3
    assert lib.carry_gdn_kv_attention(a, None) == -2
    a.HQ, a.rows.N = 4, 3
    assert lib.carry_gdn_kv_attention(a, None) == -2
    a.rows.N = a.rows.B = a.rows.max_query = 0
    assert lib.carry_gdn_kv_attention(a, None) == 0                             # nothing to do
    c.block = 48
    assert lib.carry_gdn_kv_attention(a, None) == -2
    n = _lib.NormArgs()
    assert lib.carry_gdn_add_rms_norm_quant(n, None) == -2
    n.N, n.W, n.group = 1, 8, 64
    assert lib.carry_gdn_add_rms_norm_quant(n, None) == -2
    n.group, n.W = 0, 32769
    assert lib.carry_gdn_add_rms_norm_quant(n, None) == -8
    n.W = 8
    assert lib.carry_gdn_add_rms_norm_quant(n, None) == -1


def test_oracle_scale_is_the_smallest_power_of_two():
    for amax in (448.0, 448.0001, 1.0, 3.5, 3.5001, 1e-20, 7e30):
        s = orc.power_of_two_scale(amax)
        assert amax / s <= 448 < 2 * amax / s
    assert orc.power_of_two_scale(0.0) == orc.power_of_two_scale(1e-45) == 2.0 ** -100
