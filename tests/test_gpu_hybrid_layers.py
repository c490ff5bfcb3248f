"""The example of both kinds of layer: the attention layer against a plain computation on unquantized keys and values,
and a decoded token against the same token at the end of a longer prompt."""

import os
import sys

import pytest
import torch

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
sys.path.insert(0, os.path.join(ROOT, "examples"))

pytestmark = pytest.mark.gpu


def plain_attention(layers, x, lengths):
    """Whole prompts through the attention layer in fp32, nothing in 8 bits."""
    y = x.float()
    y = y * torch.rsqrt(y.square().mean(-1, keepdim=True) + 1e-6)
    out = []
    for rows in y.split(lengths):
        h = (rows @ layers.w_qkv.float().T).view(len(rows), -1, layers.dim).transpose(0, 1)
        q, k, v = h.split([layers.heads, layers.kv_heads, layers.kv_heads])
        k, v = (t.repeat_interleave(layers.heads // layers.kv_heads, 0) for t in (k, v))
        s = (q @ k.transpose(1, 2) * layers.dim ** -0.5).masked_fill(torch.ones(len(rows), len(rows), device=x.device).triu(1).bool(), -torch.inf)
        out.append((torch.softmax(s, -1) @ v).transpose(0, 1).reshape(len(rows), -1) @ layers.w_out.float().T)
    return torch.cat(out)


def test_prompts_through_the_attention_layer():
    """e4m3 keeps 4 bits of rows, keys and values: 2^-5 of a number is a rounding's largest error, an eighth of that in
    root mean square over the sums behind an output, three roundings after one another; twice that is allowed."""
    from hybrid_layers import HybridLayers
    layers = HybridLayers(3, 200)
    lengths = [200, 1, 77]
    x = torch.randn(sum(lengths), layers.W, device="cuda", generator=torch.Generator("cuda").manual_seed(3)).bfloat16()
    layers.lengths.copy_(torch.tensor(lengths))
    start = torch.tensor([0, 200, 201, 278], dtype=torch.int32, device="cuda")
    got = layers.attention(x, torch.zeros_like(x), start, 200).float()
    want = plain_attention(layers, x, lengths)
    assert (got - want).norm() <= 2 * 3 ** 0.5 * 2.0 ** -5 * want.norm()


def test_a_decoded_token_is_the_prompts_next():
    """The cache of 60 tokens and then one more holds what that of 61 does, scales grown in a block apart: those move
    codes below e4m3's normal numbers by half a step of theirs."""
    from hybrid_layers import HybridLayers
    x = torch.randn(61, 1024, device="cuda", generator=torch.Generator("cuda").manual_seed(4)).bfloat16()
    whole, split = HybridLayers(1, 100), HybridLayers(1, 100)
    whole.lengths += 61
    want = whole.attention(x, torch.zeros_like(x))[-1:]
    split.lengths += 60
    split.attention(x[:60], torch.zeros_like(x[:60]))
    split.lengths += 1
    got = split.attention(x[60:], torch.zeros_like(x[60:]))
    assert (got.float() - want.float()).norm() <= 2.0 ** -7 * want.float().norm()


def test_steps_of_both_layers_in_a_graph(capsys):
    import hybrid_layers
    hybrid_layers.main()
    assert "finite: True" in capsys.readouterr().out
