"""The gated delta rule over whole sequences where strong decays and slow ones follow one another within a chunk."""

import math

import pytest
import torch

from oracle import prompt_oracle as orc
from test_gpu_prefill import BF16, F16, F32, bounds, goes_in_chunks, make, run

pytestmark = pytest.mark.gpu


def strong_and_slow(n, HV, seed=0):
    """Log decays by head: one of -200, -48 or -12 every third, fifth or eighth token, and -0.005 to -0.1 at the others."""
    g = torch.Generator().manual_seed(seed)
    slow = torch.exp(torch.empty(n, HV, dtype=torch.float64).uniform_(math.log(0.005), math.log(0.1), generator=g))
    t = torch.arange(n)
    for h, (every, strong) in enumerate([(3, 200.0), (5, 200.0), (8, 48.0), (5, 12.0)]):
        slow[t % every == 0, h] = strong
    return slow


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("n", [127, 191, 250])
def test_slow_decays_between_strong_ones(dtype, D, n):
    """The decay between two tokens is as good as an exponential in fp32 of what lies between them, whatever came before.

    Of the decays that count, above 2^-10, the exponent's difference is good to a few 2^-24 of at most 10, the exponential to 2^-22: 2^-20
    for an entry of L and P.  Off the diagonal entries carry a key's product with another one, less than 1, and errors are as good as
    independent: a state within 2^-20 of itself, with T in two bf16 numbers (2^-18 of an entry at most, a third of it in the mean) within 2^-19."""
    H, HV, lengths = 1, 4, [n]
    c, state = make(lengths, H, HV, D, dtype, True, gates=F32)
    x = strong_and_slow(n, HV)
    c["A_log"], c["dt_bias"] = torch.zeros(HV), torch.zeros(HV)
    c["a"] = torch.where(x > 20, x, torch.log(torch.expm1(x))).float()      # softplus of it is x
    assert goes_in_chunks(lengths, dtype)
    out, final = run(c, state, lengths, HV, D)
    wanted = orc.delta_rule(**{k: v for k, v in c.items() if k != "mixed_qkv"}, mixed=c["mixed_qkv"], H=H, D=D, lengths=lengths, initial=state)
    out_bound, state_bound = bounds(out, wanted, True, dtype == F32)
    assert ((out.cpu().double() - wanted[0]).abs() <= out_bound).all()
    off = final.cpu().double() - wanted[1]
    assert (off.abs() <= state_bound).all()
    within = 2.0 ** (-20 if dtype == F32 else -19)
    for h in range(HV):
        assert off[0, h].norm() <= within * wanted[1][0, h].norm(), f"head {h}: {off[0, h].norm() / wanted[1][0, h].norm():.2e}"
