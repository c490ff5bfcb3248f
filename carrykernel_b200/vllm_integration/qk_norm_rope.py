"""Norm and rotation of queries and keys, in one pass: what a full-attention layer does between its projections and the
key/value cache (``quantized_kv_cache``).

Every query and key head is RMS-normed over its own width, and its first numbers are rotated by angles that go with the
token's position, or, for pictures and video, with its positions on several axes (time, height, width), each of which
has some of the frequencies.  One launch reads each head once and writes it once; nothing is allocated or read back, so
the call can be captured in a CUDA graph.  carrykernel has no counterpart.  There is no CPU path.
"""

from __future__ import annotations

import torch

from .. import _lib

MAX_WIDTH = 512
MAX_AXES = 4


def _apart(t):
    """Whether no two rows of ``t [N, heads, D]`` share memory, the rows along the smaller stride lying within the larger one."""
    steps = sorted((s, n) for s, n in zip(t.stride(), t.shape[:2]) if n > 1)
    return all(s >= within for (s, _), within in zip(steps, [t.shape[2]] + [s * (n - 1) + t.shape[2] for s, n in steps]))


def qk_norm_rope(q, k, q_weight, k_weight, cos_sin, positions, eps: float = 1e-6, q_out=None, k_out=None, sections=None,
                 interleaved: bool = False, weight_offset: float = 0.0, status=None):
    """``y = x * rsqrt(mean(x ** 2) + eps) * (weight + weight_offset)`` for every head ``x`` of ``q [N, HQ, D]`` and ``k [N, HK, D]``
    (fp32, bf16 or fp16), then the rotation of ``y``; into ``q_out`` and ``k_out``, or in place where they are not given.  Returns both.

    ``cos_sin [P, R]`` holds the cosines of position ``p`` in the first ``R / 2`` columns of row ``p`` and the sines in the others; the first
    ``R <= D`` numbers of a head are rotated.  Pair ``i`` is numbers ``i`` and ``i + R / 2``, or ``2 i`` and ``2 i + 1`` with ``interleaved``.
    ``positions`` is ``[N]`` (int32 or int64), or ``[axes, N]`` with ``sections``, the number of frequencies of each axis: the first
    ``sections[0]`` go by the first axis, and so on; they add up to ``R / 2``.

    A token with a negative position is left alone; so is one with a position beyond the table, which sets
    ``STATUS_BAD_RANGE`` in ``status``.  A head with a number that is not finite becomes NaN; squares below fp32's range count as 0
    (``eps`` stands in for them).  ``q_out`` and ``k_out`` may not overlap
    ``q`` and ``k`` other than by being them."""
    lib = _lib._lib or _lib.load_library()
    if lib.native.qk_norm_rope(lib.native_table, q, k, q_weight, k_weight, cos_sin, positions, eps, q_out, k_out, sections, interleaved,
                               weight_offset, status):
        return (q if q_out is None else q_out), (k if k_out is None else k_out)
    # not a call the native path takes as it stands: the checks below say what is wrong with it, if anything
    q_out, k_out = q if q_out is None else q_out, k if k_out is None else k_out
    if q.dim() != 3 or k.dim() != 3:
        raise ValueError("q and k must be 3-D [N, heads, D]")
    N, HQ, D = q.shape
    HK = k.shape[1]
    if D == 0 or D % 2 or D > MAX_WIDTH:
        raise ValueError(f"the head width must be even and at most {MAX_WIDTH}, got {D}")
    for name, t, heads in (("q", q, HQ), ("q_out", q_out, HQ), ("k", k, HK), ("k_out", k_out, HK)):
        _lib.need_shape(t, (N, heads, D), name)
        if t.stride(-1) != 1:
            raise ValueError(f"{name} must be contiguous in its last dimension")
        if t.dtype != q.dtype:
            raise ValueError("q, k, q_out and k_out must share a dtype")
    for name, t in (("q_out", q_out), ("k_out", k_out)):
        if N and t.shape[1] and not _apart(t):
            raise ValueError(f"{name}: rows that are written must not share memory")
    for name, t in (("q_weight", q_weight), ("k_weight", k_weight)):
        _lib.need_shape(t, (D,), name)
        if not t.is_contiguous() or t.dtype != q_weight.dtype:
            raise ValueError("q_weight and k_weight must be contiguous and share a dtype")
    if cos_sin.dim() != 2 or cos_sin.shape[1] % 2 or cos_sin.shape[1] > D or (cos_sin.shape[1] > 1 and cos_sin.stride(1) != 1):
        raise ValueError(f"cos_sin must be [positions, R] with an even R of at most {D}, contiguous in its last dimension")
    if positions.dtype not in (torch.int32, torch.int64):
        raise ValueError("positions must be int32 or int64")
    half = cos_sin.shape[1] // 2
    if positions.dim() == 1 and sections is None:
        axes, sections = 1, [half]
    else:
        axes = positions.shape[0] if positions.dim() == 2 else 1
        if sections is None or len(sections) != axes or not 1 <= axes <= MAX_AXES:
            raise ValueError(f"positions must be [N], or [axes, N] with as many sections and at most {MAX_AXES} axes")
        sections = [int(s) for s in sections]
        if min(sections) < 0 or sum(sections) != half:
            raise ValueError(f"sections must add up to the {half} frequencies of cos_sin, got {sections}")
    _lib.need_shape(positions, (axes, N) if positions.dim() == 2 else (N,), "positions")
    if N > 1 and positions.stride(-1) != 1:
        raise ValueError("positions must be contiguous in their last dimension")
    if not float(eps) >= 0.0:
        raise ValueError(f"eps must not be negative, got {eps}")
    dev = q.device
    _lib.same_device(dev, k=k, q_out=q_out, k_out=k_out, q_weight=q_weight, k_weight=k_weight, cos_sin=cos_sin, positions=positions)
    a = _lib.RotateArgs()
    a.status = _lib.status_ptr(status, dev)
    a.q, a.k, a.q_out, a.k_out = q.data_ptr(), k.data_ptr(), q_out.data_ptr(), k_out.data_ptr()
    a.stride_q_tok, a.stride_q_head, a.stride_k_tok, a.stride_k_head = q.stride(0), q.stride(1), k.stride(0), k.stride(1)
    a.stride_q_out_tok, a.stride_q_out_head = q_out.stride(0), q_out.stride(1)
    a.stride_k_out_tok, a.stride_k_out_head = k_out.stride(0), k_out.stride(1)
    a.q_weight, a.k_weight, a.weight_dtype = q_weight.data_ptr(), k_weight.data_ptr(), _lib.dtype_id(q_weight)
    a.cos_sin, a.stride_table, a.table_rows, a.table_dtype = cos_sin.data_ptr(), cos_sin.stride(0), cos_sin.shape[0], _lib.dtype_id(cos_sin)
    a.positions, a.positions_64 = positions.data_ptr(), int(positions.dtype == torch.int64)
    a.stride_positions = positions.stride(0) if positions.dim() == 2 else 0
    a.eps, a.weight_offset, a.interleaved, a.dtype = float(eps), float(weight_offset), int(bool(interleaved)), _lib.dtype_id(q)
    a.N, a.HQ, a.HK, a.D, a.rotary, a.axes = N, HQ, HK, D, 2 * half, axes
    for i, s in enumerate(sections):
        a.sections[i] = s
    _lib.require_cuda(q, "q")
    with torch.cuda.device(dev):
        rc = lib.carry_gdn_qk_norm_rope(a, _lib.current_stream_ptr(dev))
    _lib.check(rc, "carry_gdn_qk_norm_rope")
    return q_out, k_out
