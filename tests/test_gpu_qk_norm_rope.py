"""Norm and rotation of queries and keys against the definitions in 64 bits."""

import pytest
import torch

from carrykernel_b200 import _lib
from carrykernel_b200.vllm_integration.qk_norm_rope import qk_norm_rope
from oracle import prompt_oracle as orc

pytestmark = pytest.mark.gpu

BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32
DEV = "cuda"


def make(N, HQ, HK, D, R, dtype, axes=1, seed=0, P=500, table=F32):
    g = torch.Generator().manual_seed(seed)
    qkv = (torch.randn(N, HQ + 2 * HK, D, generator=g) * 3).to(dtype)
    angle = torch.arange(P, dtype=torch.float64)[:, None] * 1e4 ** (-torch.arange(0, R, 2, dtype=torch.float64) / max(R, 1))
    cos_sin = torch.cat([angle.cos(), angle.sin()], 1).to(table)
    positions = torch.randint(0, P, (N,) if axes == 1 else (axes, N), generator=g)
    weights = [torch.randn(D, generator=g).to(dtype) for _ in range(2)]
    return qkv, *weights, cos_sin, positions


def check(got, x, weight, cos_sin, positions, eps=1e-6, rows=None, **more):
    """fp32 arithmetic: a sum of squares in at most 23 additions, its root, three products and a rotation of two, 24 roundings of
    2^-24 at most relative to the pair; then one rounding to the output's type."""
    want, size = orc.qk_norm_rope(x, weight, cos_sin, positions, eps, **more)
    half_step = torch.finfo(got.dtype).eps / 2
    bound = 24 * 2.0 ** -24 * size + half_step * (want.abs() + 2.0 ** -20 * size) + torch.finfo(got.dtype).smallest_normal * half_step
    off = (got.cpu().double() - want).abs()
    assert (off <= bound if rows is None else (off <= bound)[rows]).all(), f"off by up to {(off / bound).max():.2f} of the bound"


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("N,HQ,HK,D,R,axes,interleaved", [
    (1, 32, 8, 128, 128, 1, False), (7, 16, 2, 128, 32, 1, False), (65, 4, 4, 64, 64, 1, True), (3, 5, 1, 96, 48, 1, False),
    (130, 3, 3, 256, 64, 3, False), (9, 2, 1, 512, 512, 1, False), (4, 2, 2, 512, 256, 4, True), (5, 3, 1, 128, 0, 1, False),
    (6, 3, 2, 6, 4, 1, False), (6, 3, 2, 6, 2, 1, True), (11, 2, 1, 80, 20, 2, False), (2, 1, 1, 2, 2, 1, False), (1500, 8, 2, 128, 128, 3, False)])
def test_against_definition(dtype, N, HQ, HK, D, R, axes, interleaved):
    qkv, qw, kw, cos_sin, positions = make(N, HQ, HK, D, R, dtype, axes)
    q, k, v = qkv.split([HQ, HK, HK], dim=1)
    sections = None
    if axes > 1:
        sections = [R // 2 // axes] * axes
        sections[0] += R // 2 - sum(sections)
    dq, dk, _ = qkv.to(DEV).split([HQ, HK, HK], dim=1)
    q_out, k_out = torch.empty(N, HQ, D, dtype=dtype, device=DEV), torch.empty(N, HK, D, dtype=dtype, device=DEV)
    got = qk_norm_rope(dq, dk, qw.to(DEV), kw.to(DEV), cos_sin.to(DEV), positions.to(DEV), q_out=q_out, k_out=k_out, sections=sections,
                       interleaved=interleaved)
    assert got[0] is q_out and got[1] is k_out
    check(q_out, q, qw, cos_sin, positions, sections=sections, interleaved=interleaved)
    check(k_out, k, kw, cos_sin, positions, sections=sections, interleaved=interleaved)
    if N * D < 50000:
        assert _lib.load_library().carry_gdn_last_kernel() == 12


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("shift", [0, 1, 2])
def test_in_place_on_rows_of_any_alignment(dtype, shift):
    """In place, in a wider row that begins off the grid; the values beside them stay as they were."""
    N, HQ, HK, D = 9, 3, 2, 64
    qkv, qw, kw, cos_sin, positions = make(N, HQ, HK, D, 32, dtype)
    wide = torch.full((N, (HQ + 2 * HK) * D + 5), 7.0, dtype=dtype)
    wide[:, shift:shift + (HQ + 2 * HK) * D] = qkv.flatten(1)
    dev = wide.to(DEV)
    q, k, _ = dev[:, shift:shift + (HQ + 2 * HK) * D].unflatten(1, (HQ + 2 * HK, D)).split([HQ, HK, HK], dim=1)
    qk_norm_rope(q, k, qw.to(DEV), kw.to(DEV), cos_sin.to(DEV), positions.int().to(DEV))
    check(q, qkv[:, :HQ], qw, cos_sin, positions)
    check(k, qkv[:, HQ:HQ + HK], kw, cos_sin, positions)
    same = torch.ones_like(wide, dtype=torch.bool)
    same[:, shift:shift + (HQ + HK) * D] = False
    assert torch.equal(dev.cpu()[same], wide[same])


def test_positions_outside_the_table():
    N, D = 6, 64
    qkv, qw, kw, cos_sin, _ = make(N, 2, 1, D, D, BF16)
    positions = torch.tensor([3, -1, 499, 500, 2 ** 40, 0])
    q, k = qkv[:, :2].to(DEV), qkv[:, 2:3].to(DEV)
    q_out, k_out = torch.full_like(q, 5.0), torch.full_like(k, 5.0)
    status = torch.zeros(1, dtype=torch.int32, device=DEV)
    qk_norm_rope(q, k, qw.to(DEV), kw.to(DEV), cos_sin.to(DEV), positions.to(DEV), q_out=q_out, k_out=k_out, status=status)
    rows = torch.tensor([0, 2, 5])
    check(q_out, qkv[:, :2], qw, cos_sin, positions, rows=rows)
    check(k_out, qkv[:, 2:3], kw, cos_sin, positions, rows=rows)
    assert (q_out[[1, 3, 4]] == 5).all() and (k_out[[1, 3, 4]] == 5).all()
    assert status.item() == _lib.STATUS_BAD_RANGE
    status.zero_()
    qk_norm_rope(q[:3], k[:3], qw.to(DEV), kw.to(DEV), cos_sin.to(DEV), positions[:3].to(DEV), q_out=q_out[:3], k_out=k_out[:3], status=status)
    assert status.item() == 0                            # a negative position is padding


def test_weight_offset_eps_and_tables_of_other_types():
    N, HQ, HK, D = 5, 2, 2, 128
    for table in (F16, BF16):
        qkv, qw, kw, cos_sin, positions = make(N, HQ, HK, D, D, F16, table=table)
        q, k = qkv[:, :HQ].to(DEV), qkv[:, HQ:HQ + HK].to(DEV)
        out = torch.empty_like(q), torch.empty_like(k)
        qk_norm_rope(q, k, qw.float().to(DEV), kw.float().to(DEV), cos_sin.to(DEV), positions.to(DEV), 0.25, *out, weight_offset=1.0)
        check(out[0], qkv[:, :HQ], qw, cos_sin, positions, eps=0.25, offset=1.0)
        check(out[1], qkv[:, HQ:HQ + HK], kw, cos_sin, positions, eps=0.25, offset=1.0)


def test_values_at_the_end_of_the_range_and_not_finite():
    D = 128
    qkv, qw, kw, cos_sin, positions = make(6, 2, 1, D, 64, F32)
    x = qkv[:, :2].clone()
    x[0] *= 1e37
    x[1, 0, 5], x[2, 1, 100], x[3, 0, 0] = float("inf"), float("nan"), -3e38
    x[4] = 0.0
    k = qkv[:, 2:3]
    out = torch.empty(6, 2, D, device=DEV), torch.empty(6, 1, D, device=DEV)
    qk_norm_rope(x.to(DEV), k.to(DEV), qw.to(DEV), kw.to(DEV), cos_sin.to(DEV), positions.to(DEV), q_out=out[0], k_out=out[1])
    bad = torch.zeros(6, 2, dtype=torch.bool)
    bad[1, 0] = bad[2, 1] = True
    assert out[0].cpu().isnan().all(-1).equal(bad) and not out[0].cpu()[~bad].isnan().any()
    x[bad] = 1.0
    check(torch.where(bad[..., None].to(DEV), 0.0, out[0]), x, qw, cos_sin, positions, rows=torch.tensor([0, 3, 4, 5]))
    check(out[1], k, kw, cos_sin, positions)


def test_captured_and_replayed_on_another_stream():
    N, HQ, HK, D = 33, 4, 2, 128
    qkv, qw, kw, cos_sin, positions = make(N, HQ, HK, D, D, BF16)
    q, k = qkv[:, :HQ].to(DEV), qkv[:, HQ:HQ + HK].to(DEV)
    out = torch.empty_like(q), torch.empty_like(k)
    rest = (qw.to(DEV), kw.to(DEV), cos_sin.to(DEV))
    p = positions.to(DEV)
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        qk_norm_rope(q, k, *rest, p, q_out=out[0], k_out=out[1])
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        qk_norm_rope(q, k, *rest, p, q_out=out[0], k_out=out[1])
    p.copy_((positions + 17) % 500)
    q.mul_(2)
    graph.replay()
    torch.cuda.synchronize()
    check(out[0], qkv[:, :HQ] * 2, qw, cos_sin, (positions + 17) % 500)
    check(out[1], qkv[:, HQ:HQ + HK], kw, cos_sin, (positions + 17) % 500)


def test_one_axis_in_a_row_of_its_own_needs_its_section():
    N, HQ, HK, D = 9, 2, 1, 64
    qkv, qw, kw, cos_sin, positions = make(N, HQ, HK, D, D, BF16)
    q, k = qkv[:, :HQ].to(DEV), qkv[:, HQ:HQ + HK].to(DEV)
    rest = (qw.to(DEV), kw.to(DEV), cos_sin.to(DEV), positions.to(DEV)[None])
    out = torch.empty_like(q), torch.empty_like(k)
    with pytest.raises(ValueError):
        qk_norm_rope(q, k, *rest, q_out=out[0], k_out=out[1])
    qk_norm_rope(q, k, *rest, q_out=out[0], k_out=out[1], sections=[D // 2])
    check(out[0], qkv[:, :HQ], qw, cos_sin, positions)
    check(out[1], qkv[:, HQ:HQ + HK], kw, cos_sin, positions)


def test_numbers_whose_squares_are_below_fp32():
    """eps stands in for them: numbers come out by their weight over eps's root."""
    N, HQ, HK, D = 3, 2, 1, 128
    qkv, qw, kw, cos_sin, positions = make(N, HQ, HK, D, D, F32)
    qkv = qkv * 1e-25
    q, k = qkv[:, :HQ].to(DEV), qkv[:, HQ:HQ + HK].to(DEV)
    qk_norm_rope(q, k, qw.to(DEV), kw.to(DEV), cos_sin.to(DEV), positions.to(DEV))
    check(q, qkv[:, :HQ], qw, cos_sin, positions)
    check(k, qkv[:, HQ:HQ + HK], kw, cos_sin, positions)


@pytest.mark.parametrize("shift", [0, 1])
def test_offsets_beyond_32_bits(shift):
    """Rows and table rows that lie more than 2^31 numbers apart."""
    N, HQ, HK, D, stride = 70, 3, 2, 64, 2 ** 25 + shift
    qkv, qw, kw, cos_sin, positions = make(N, HQ, HK, D, D, BF16, P=N)
    buffer = torch.empty(N * stride, dtype=BF16, device=DEV)
    q, k = buffer.as_strided((N, HQ, D), (stride, D, 1)), buffer.as_strided((N, HK, D), (stride, D, 1), 512)
    table = torch.empty(N * stride, device=DEV).as_strided((N, D), (stride, 1))
    q.copy_(qkv[:, :HQ]), k.copy_(qkv[:, HQ:HQ + HK]), table.copy_(cos_sin)
    positions[0] = N - 1
    qk_norm_rope(q, k, qw.to(DEV), kw.to(DEV), table, positions.to(DEV))
    check(q, qkv[:, :HQ], qw, cos_sin, positions)
    check(k, qkv[:, HQ:HQ + HK], kw, cos_sin, positions)
