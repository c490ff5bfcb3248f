"""The workspace of the key/value attention is as large as the cache's own device asks for, whichever one is current: the number of
its processors decides how contexts are cut."""

import contextlib
import types

import torch

from carrykernel_b200 import _lib
from carrykernel_b200.vllm_integration import quantized_kv_cache as qkv


def test_asked_for_on_the_device_of_the_cache(monkeypatch):
    current = ["another"]
    cache = qkv.init_quantized_kv(5, 2, 64, 128, "cpu")

    @contextlib.contextmanager
    def device_of(tensor):
        before, current[0] = current[0], "the cache's" if tensor is cache[0] else "another"
        yield
        current[0] = before

    monkeypatch.setattr(torch.cuda, "device_of", device_of)
    monkeypatch.setattr(_lib, "_lib", types.SimpleNamespace(
        carry_gdn_kv_attention_workspace=lambda args: 4096 if current[0] == "the cache's" else 0))
    q, table = torch.zeros(3, 4, 128), torch.zeros(3, 2, dtype=torch.int32)
    assert qkv.attention_workspace_bytes(q, cache[0], cache[1], table) == 4096
    assert current[0] == "another"
