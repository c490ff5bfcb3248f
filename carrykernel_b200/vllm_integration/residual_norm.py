"""The entry of a decoder layer: residual addition, RMS norm, and the normed row in 8 bits with its scales.

Both kinds of layer of a hybrid model (Gated DeltaNet and full attention) begin with it, and so does the feed-forward
part: the projections behind it take e4m3 rows with a scale per token, or per 128 columns.  One launch reads ``x`` and
the residual once and writes the new residual, the codes and the scales; nothing is allocated or read back, so the
call can be captured in a CUDA graph.  There is no CPU path.
"""

from __future__ import annotations

import torch

from .. import _lib

CODES = torch.float8_e4m3fn
GROUP = 128
MAX_WIDTH = 32768


def _row_matrix(t, shape, name):
    _lib.need_shape(t, shape, name)
    if t.stride(1) != 1 and shape[1] > 1:
        raise ValueError(f"{name} must be contiguous in its last dimension")


def add_rms_norm_quant(x, residual, weight, codes, scale, eps: float = 1e-6, residual_out=None):
    """``h = x + residual`` in fp32, ``residual_out = h``, ``y = h * rsqrt(mean(h ** 2) + eps) * weight``, and ``y``
    as ``codes * scale``; returns ``(codes, scale)``.

    ``x``, ``residual`` ``[N, W]`` (fp32, bf16 or fp16 each, row strides free), ``weight [W]``, ``codes [N, W]``
    float8_e4m3fn, ``scale`` fp32: ``[N]`` for one scale per row or ``[N, ceil(W / 128)]`` for one per 128 columns.
    ``scale = max(amax|y|, 1e-12) / 448``.  The sum goes back into ``residual`` unless ``residual_out`` (its dtype) is
    given; with ``residual=None`` (a model's first layer) ``h = x``, stored only where ``residual_out`` is given.  A row
    of ``h`` with a number that is not finite, or whose product with its weight is not in fp32, gets NaN codes and scales."""
    lib = _lib._lib or _lib.load_library()
    if lib.native.add_rms_norm(lib.native_table, x, residual, weight, codes, scale, eps, residual_out):
        return codes, scale
    if x.dim() != 2:
        raise ValueError(f"x must be 2-D [N, W], got {tuple(x.shape)}")
    N, W = x.shape
    if W == 0 or W > MAX_WIDTH:
        raise ValueError(f"the row width must be 1 to {MAX_WIDTH}, got {W}")
    if residual_out is None:
        residual_out = residual
    _row_matrix(x, (N, W), "x")
    for name, t in (("residual", residual), ("residual_out", residual_out)):
        if t is not None:
            _row_matrix(t, (N, W), name)
    if residual is not None and residual.dtype != residual_out.dtype:
        raise ValueError("residual and residual_out must share a dtype")
    _row_matrix(codes, (N, W), "codes")
    if codes.dtype != CODES:
        raise ValueError("codes must be float8_e4m3fn")
    _lib.need_shape(weight, (W,), "weight")
    groups = -(-W // GROUP)
    if scale.dtype != torch.float32 or not scale.is_contiguous() or tuple(scale.shape) not in ((N,), (N, groups)):
        raise ValueError(f"scale must be a contiguous fp32 [{N}] or [{N}, {groups}], got {scale.dtype} {tuple(scale.shape)}")
    if not weight.is_contiguous():
        raise ValueError("weight must be contiguous")
    dev = x.device
    _lib.same_device(dev, residual=residual, residual_out=residual_out, weight=weight, codes=codes, scale=scale)
    _lib.require_cuda(x, "x")
    a = _lib.NormArgs()
    a.x, a.stride_x, a.x_dtype = x.data_ptr(), x.stride(0), _lib.dtype_id(x)
    a.residual_dtype = a.x_dtype
    if residual is not None:
        a.residual, a.stride_residual, a.residual_dtype = residual.data_ptr(), residual.stride(0), _lib.dtype_id(residual)
    if residual_out is not None:
        a.residual_out, a.stride_residual_out = residual_out.data_ptr(), residual_out.stride(0)
        a.residual_dtype = _lib.dtype_id(residual_out)
    a.weight, a.weight_dtype = weight.data_ptr(), _lib.dtype_id(weight)
    a.codes, a.stride_codes, a.scale = codes.data_ptr(), codes.stride(0), scale.data_ptr()
    a.eps, a.N, a.W, a.group = float(eps), N, W, GROUP if scale.dim() == 2 else 0
    with torch.cuda.device(dev):
        rc = lib.carry_gdn_add_rms_norm_quant(a, _lib.current_stream_ptr(dev))
    _lib.check(rc, "carry_gdn_add_rms_norm_quant")
    return codes, scale
