"""Two decoder layers of a hybrid model on 8-bit serving memory: a Gated-DeltaNet layer on the quantized slot pool and a
full-attention layer on the 8-bit key/value cache, each entered through the norm with 8-bit output.

``python examples/hybrid_layers.py`` takes a prompt through the attention layer in one chunk, then decodes tokens through
both layers in a captured CUDA graph, and prints the time of a step.  Weights are random; the projections are plain
matrix products of the normed rows' values (an engine would hand codes and scales to an 8-bit product).
"""

from __future__ import annotations

import os
import sys

import torch

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))
from carrykernel_b200.vllm_integration import quantized_kv_cache as qkv  # noqa: E402
from carrykernel_b200.vllm_integration import quantized_packed_decode as qpd  # noqa: E402
from carrykernel_b200.vllm_integration.residual_norm import add_rms_norm_quant  # noqa: E402
from carrykernel_b200.vllm_integration.state_cache import SlotCache  # noqa: E402


class HybridLayers:
    """One recurrent and one attention layer of width ``W`` for up to ``requests`` requests of ``tokens`` tokens."""

    def __init__(self, requests, tokens, W=1024, heads=8, kv_heads=2, dim=128, page=64, block=32, device="cuda", seed=0):
        g = torch.Generator(device=device).manual_seed(seed)
        new = lambda *shape: (torch.randn(shape, device=device, generator=g) * shape[-1] ** -0.5).bfloat16()  # noqa: E731
        self.requests, self.W, self.heads, self.kv_heads, self.dim, self.page = requests, W, heads, kv_heads, dim, page
        self.w_norm = torch.ones(2, W, dtype=torch.bfloat16, device=device)
        # recurrent layer: q, k, v and the two gates out of the row
        self.w_mixed, self.w_gates, self.w_out_gdn = new(3 * heads * dim, W), new(2 * heads, W), new(W, heads * dim)
        self.A_log, self.dt_bias = torch.zeros(heads, device=device), torch.zeros(heads, device=device)
        self.slots = SlotCache(1, requests + 1, heads, dim, dim, device)
        for r in range(requests):
            self.slots.allocate(r)
        self.slot_ids = self.slots.indices(range(requests))
        # attention layer; pages are handed out in order here, page 0 being the padding page
        self.w_qkv, self.w_out = new((heads + 2 * kv_heads) * dim, W), new(W, heads * dim)
        per = -(-tokens // page)
        self.cache = qkv.init_quantized_kv(requests * per + 1, kv_heads, page, dim, device, block=block)
        self.table = torch.arange(1, requests * per + 1, dtype=torch.int32, device=device).view(requests, per)
        self.lengths = torch.zeros(requests, dtype=torch.int32, device=device)

    def normed(self, x, residual, layer):
        """The layer's entry; the values that the 8-bit rows stand for.  ``residual`` becomes the sum."""
        codes = torch.empty(x.shape, dtype=torch.float8_e4m3fn, device=x.device)
        scale = torch.empty(x.shape[0], -(-self.W // 128), device=x.device)
        add_rms_norm_quant(x, residual, self.w_norm[layer], codes, scale)
        return (codes.float() * scale.repeat_interleave(128, dim=1)[:, :self.W]).bfloat16()

    def recurrent(self, x, residual):
        """One token of every request through the Gated-DeltaNet layer."""
        y = self.normed(x, residual, 0)
        a, b = (y @ self.w_gates.T).view(-1, 2, self.heads).unbind(1)
        out = torch.empty(self.requests, 1, self.heads, self.dim, dtype=torch.bfloat16, device=x.device)
        qpd.quantized_gated_delta_rule_packed_decode(
            y @ self.w_mixed.T, a, b, self.A_log, self.dt_bias, self.dim ** -0.5, *self.slots.pools[0], out, self.slot_ids,
            use_qk_l2norm_in_kernel=True, resid_fmt=self.slots.resid_fmt)
        return out.view(self.requests, -1) @ self.w_out_gdn.T

    def attention(self, x, residual, query_start=None, max_query_len=None):
        """New tokens through the attention layer: into the cache, then over it.  ``lengths`` already counts them."""
        y = self.normed(x, residual, 1)
        q, k, v = (y @ self.w_qkv.T).view(-1, self.heads + 2 * self.kv_heads, self.dim).split([self.heads, self.kv_heads, self.kv_heads], dim=1)
        more = dict(query_start=query_start, max_query_len=max_query_len)
        qkv.quantized_kv_append(k, v, *self.cache, self.table, self.lengths, **more)
        out = torch.empty(q.shape, dtype=q.dtype, device=q.device)
        qkv.quantized_paged_attention(q, self.dim ** -0.5, *self.cache, out, self.table, self.lengths, **more)
        return out.view(x.shape[0], -1) @ self.w_out.T

    def step(self, x, residual):
        """One decoded token of every request through both layers."""
        self.lengths += 1
        return self.attention(self.recurrent(x, residual), residual)


def main():
    B, prompt = 16, 1000
    layers = HybridLayers(B, prompt + 200)
    x = torch.randn(B * prompt, layers.W, device="cuda").bfloat16()
    layers.lengths += prompt
    layers.attention(x, torch.zeros_like(x))
    x = x.view(B, prompt, -1)[:, -1].contiguous()
    residual = torch.zeros_like(x)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        layers.step(x, residual)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = layers.step(x, residual)
    start, end = (torch.cuda.Event(enable_timing=True) for _ in range(2))
    start.record()
    for _ in range(100):
        graph.replay()
    end.record()
    torch.cuda.synchronize()
    print(f"{B} requests, contexts of {int(layers.lengths[0])} tokens: {start.elapsed_time(end) * 10:.1f} us a step of both layers; "
          f"finite: {bool(y.isfinite().all())}")


if __name__ == "__main__":
    main()
