"""A prompt's way through the example's layers, as a run of calls: norm, recurrence over the sequence, state into the slots; norm, rotation,
append, attention.  Against plain computations, and a decoded token against the same token at the end of a longer prompt."""

import os
import sys

import pytest
import torch

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
sys.path.insert(0, os.path.join(ROOT, "examples"))

pytestmark = pytest.mark.gpu


def rows(n, seed):
    return torch.randn(n, 1024, device="cuda", generator=torch.Generator("cuda").manual_seed(seed)).bfloat16()


def test_a_decoded_token_is_the_prompts_next_in_the_recurrent_layer():
    """The state goes through int8 codes with an int4 residual: a number is off by 1 / (127 * 14) of its row's largest at most, and the
    token decays and adds to it alike, so that its output is off by that of the state's part in it; the rows' own roundings (8-bit
    rows with a scale of their own, bf16 products and outputs) are the same on both sides but for the output's, 2^-8."""
    from hybrid_layers import HybridLayers
    for n in (40, 161):
        x = rows(n + 1, n)
        whole, split = HybridLayers(1, 10), HybridLayers(1, 10)
        want = whole.recurrent_prompt(x, torch.zeros_like(x))[-1:]
        split.recurrent_prompt(x[:n], torch.zeros_like(x[:n]))
        got = split.recurrent(x[n:], torch.zeros_like(x[n:]))
        assert (got.float() - want.float()).norm() <= 2.0 ** -6 * want.float().norm()


def test_ragged_prompts_are_prompts_alone():
    from hybrid_layers import HybridLayers
    lengths = [100, 1, 77]
    x = rows(sum(lengths), 5)
    start = torch.tensor([0, 100, 101, 178], dtype=torch.int32, device="cuda")
    together = HybridLayers(3, 100, rotate=True)
    together.lengths.copy_(torch.tensor(lengths))
    residual = torch.zeros_like(x)
    got = together.attention(together.recurrent_prompt(x, residual, start, 100), residual, start, 100)
    for i, n in enumerate(lengths):
        part = x[start[i]:start[i] + n]
        alone = HybridLayers(1, 100, rotate=True)
        alone.lengths += n
        residual = torch.zeros_like(part)
        want = alone.attention(alone.recurrent_prompt(part, residual), residual)
        # other tilings of the plain matrix products and of the attention: bf16 roundings that fall the other way, and 8-bit codes with them
        assert (got[start[i]:start[i] + n].float() - want.float()).norm() <= 2.0 ** -4 * want.float().norm()


def test_rotated_attention_over_prompts():
    """As the attention layer without rotation is tested: e4m3 keeps 4 bits of rows, keys and values."""
    from hybrid_layers import HybridLayers
    layers = HybridLayers(2, 150, rotate=True)
    lengths = [150, 60]
    x = rows(sum(lengths), 6)
    layers.lengths.copy_(torch.tensor(lengths))
    start = torch.tensor([0, 150, 210], dtype=torch.int32, device="cuda")
    got = layers.attention(x, torch.zeros_like(x), start, 150).float()
    y = x.float()
    y = y * torch.rsqrt(y.square().mean(-1, keepdim=True) + 1e-6)
    out = []
    for part in y.split(lengths):
        h = (part @ layers.w_qkv.float().T).view(len(part), -1, layers.dim).transpose(0, 1)
        q, k, v = h.split([layers.heads, layers.kv_heads, layers.kv_heads])
        turned = []
        for z in (q, k):
            z = z * torch.rsqrt(z.square().mean(-1, keepdim=True) + 1e-6)
            cos, sin = layers.angles[:len(part)].split(layers.dim // 4, dim=1)
            one, two, rest = z.split([layers.dim // 4, layers.dim // 4, layers.dim // 2], dim=-1)
            turned.append(torch.cat([one * cos - two * sin, two * cos + one * sin, rest], -1))
        q, (k, v) = turned[0], (t.repeat_interleave(layers.heads // layers.kv_heads, 0) for t in (turned[1], v))
        s = (q @ k.transpose(1, 2) * layers.dim ** -0.5).masked_fill(torch.ones(len(part), len(part), device=x.device).triu(1).bool(), -torch.inf)
        out.append((torch.softmax(s, -1) @ v).transpose(0, 1).reshape(len(part), -1) @ layers.w_out.float().T)
    want = torch.cat(out)
    assert (got - want).norm() <= 2 * 3 ** 0.5 * 2.0 ** -5 * want.norm()
