"""The layer norm with 8-bit output on the GPU, against its definition in 64 bits."""

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


def call(x, r, w, grouped, eps=1e-6, r_out=None):
    from carrykernel_b200.vllm_integration.residual_norm import add_rms_norm_quant
    N, W = x.shape
    codes = torch.empty(N, W, dtype=torch.float8_e4m3fn, device=DEV)
    scale = torch.empty((N, -(-W // 128)) if grouped else (N,), device=DEV)
    add_rms_norm_quant(x, r, w, codes, scale, eps, residual_out=r_out)
    torch.cuda.synchronize()
    return codes, scale


def check(x, r, w, grouped, codes, scale, eps=1e-6):
    """A scale is within 2^-20 (the sum of squares, a root and a quotient in fp32); a code is e4m3's nearest of the
    exact quotient, or its neighbour where the quotient is within 2^-18 of a tie."""
    _, y, s = orc.add_rms_norm(x.cpu(), None if r is None else r.cpu(), w.cpu(), eps, 128 if grouped else 0)
    got = scale.cpu().double().view(s.shape)
    assert ((got - s).abs() <= 2.0 ** -20 * s).all()
    t = y / (s.repeat_interleave(128, 1)[:, :y.shape[1]] if grouped else s)
    half = 2.0 ** (torch.floor(torch.log2(t.abs().clamp(min=2.0 ** -6))) - 4)
    assert ((codes.cpu().float().double() - t).abs() <= half + 2.0 ** -18 * t.abs()).all()


@pytest.mark.parametrize("grouped", [False, True])
@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("N,W", [(1, 1), (3, 7), (2, 127), (5, 128), (4, 129), (7, 1000), (1, 4096), (33, 4104), (2, 8200), (3, 16384), (2, 20001), (1, 32768)])
def test_against_the_definition(N, W, dtype, grouped):
    g = torch.Generator().manual_seed(N * W)
    dt = TYPES[dtype]
    x, r = (torch.randn(N, W, generator=g) * s for s in (1.0, 3.0))
    x, r, w = x.to(dt).to(DEV), r.to(dt).to(DEV), (1 + 0.1 * torch.randn(W, generator=g)).to(dt).to(DEV)
    before, want = r.clone(), (x.float() + r.float()).to(dt)
    codes, scale = call(x, r, w, grouped)
    check(x, before, w, grouped, codes, scale)
    assert torch.equal(r, want)                          # in place


def test_types_of_x_residual_and_weight_are_independent():
    g = torch.Generator().manual_seed(5)
    x, r, w = torch.randn(9, 520, generator=g).bfloat16().to(DEV), torch.randn(9, 520, generator=g).to(DEV), torch.randn(520, generator=g).half().to(DEV)
    out = torch.zeros_like(r)
    codes, scale = call(x, r, w, True, r_out=out)
    check(x, r, w, True, codes, scale)
    assert torch.equal(out, x.float() + r)


@pytest.mark.parametrize("keep", [False, True])
def test_without_a_residual(keep):
    x, w = torch.randn(4, 640, device=DEV).half(), torch.ones(640, device=DEV)
    out = torch.zeros_like(x) if keep else None
    codes, scale = call(x, None, w, False, r_out=out)
    check(x, None, w, False, codes, scale)
    assert out is None or torch.equal(out, x)


@pytest.mark.parametrize("shift", [0, 1, 3])
def test_row_strides_and_alignment(shift):
    """Rows of a wider matrix, starting off the 16-byte boundaries."""
    g = torch.Generator().manual_seed(9)
    wide = [torch.randn(6, 700, generator=g).bfloat16().to(DEV) for _ in range(2)]
    x, r = (t[:, shift:shift + 512] for t in wide)
    guard = wide[1].clone()
    w = torch.ones(512, dtype=torch.bfloat16, device=DEV)
    before = r.clone()
    codes, scale = call(x, r, w, True)
    check(x, before, w, True, codes, scale)
    assert torch.equal(wide[1][:, :shift], guard[:, :shift]) and torch.equal(wide[1][:, shift + 512:], guard[:, shift + 512:])


def test_zero_rows_large_and_small_numbers():
    x = torch.zeros(5, 256, device=DEV)
    x[1] = 1e-30
    x[2] = 3e18
    x[3, 7] = 1e15
    w = torch.ones(256, device=DEV)
    codes, scale = call(x, torch.zeros_like(x), w, False)
    check(x, None, w, False, codes, scale)
    assert (codes[0].float() == 0).all() and scale[0].item() == pytest.approx(1e-12 / 448)


def test_rows_that_are_not_finite_are_nan_and_others_are_not():
    x = torch.randn(6, 300, device=DEV)
    x[1, 5], x[3, 299], x[4, 0] = math.nan, math.inf, -math.inf
    w = torch.ones(300, device=DEV)
    for grouped in (False, True):
        codes, scale = call(x, None, w, grouped)
        bad = torch.tensor([False, True, False, True, True, False], device=DEV)
        assert codes.float().isnan().all(1).equal(bad) and scale.view(6, -1).isnan().all(1).equal(bad)
        assert scale.view(6, -1).isfinite().all(1).equal(~bad)


def test_captured_in_a_graph_and_on_another_stream():
    x, r, w = torch.randn(16, 1024, device=DEV).bfloat16(), torch.randn(16, 1024, device=DEV).bfloat16(), torch.ones(1024, device=DEV).bfloat16()
    out = torch.zeros_like(r)
    want, want_scale = call(x, r, w, False, r_out=out)
    codes, scale = torch.zeros_like(want), torch.zeros_like(want_scale)
    from carrykernel_b200.vllm_integration.residual_norm import add_rms_norm_quant
    stream = torch.cuda.Stream()
    with torch.cuda.stream(stream):
        add_rms_norm_quant(x, r, w, codes, scale, residual_out=out)
    stream.synchronize()
    assert torch.equal(codes.view(torch.uint8), want.view(torch.uint8))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        add_rms_norm_quant(x, r, w, codes, scale, residual_out=out)
    codes.zero_(), scale.zero_()
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(codes.view(torch.uint8), want.view(torch.uint8)) and torch.equal(scale, want_scale)


def test_no_rows():
    codes, scale = call(torch.zeros(0, 64, device=DEV), torch.zeros(0, 64, device=DEV), torch.ones(64, device=DEV), True)
    assert codes.shape == (0, 64) and scale.shape == (0, 1)
