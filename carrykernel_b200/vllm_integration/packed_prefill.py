"""The gated delta rule over whole sequences: a prompt's way through a recurrent layer.

The slot-indexed decode step (``quantized_packed_decode``) advances requests by single tokens on a quantized state.  A
prompt goes ahead of it: :func:`gated_delta_rule_packed_prefill` takes the same rows, gates and head map, over every token of
ragged sequences, from a floating-point state (or none) to a floating-point state, which
``state_pool.store_state`` then quantises into the requests' slots.  For a further chunk of a prompt,
``state_pool.load_state`` hands the state back.  Few tokens go token by token, prompts in chunks of 64 on the tensor cores.

carrykernel has no prefill; the recurrence is that of its decode step
(``vllm_integration/quantized_packed_decode.py:160-200``) with the state left unquantized.

The call reads nothing back to the host, never synchronises and can be captured in a CUDA graph.  There is no CPU path.
"""

from __future__ import annotations

import torch

from .. import _lib

HEAD_DIMS = (64, 128)


def _state(t, shape, name):
    _lib.need_shape(t, shape, name)
    if t.dtype != torch.float32 or t.stride()[1:] != (shape[2] * shape[3], shape[3], 1):
        raise ValueError(f"{name} must be fp32 and dense within a request (only the request stride may vary)")
    if t.data_ptr() % 16 or t.stride(0) % 4:
        raise ValueError(f"{name}: every request's state must start on a 16-byte boundary")


def _prefill_sizes(mixed_qkv, final_state, query_start, max_query_len):
    """An argument block with a call's sizes, which is all that its workspace goes by."""
    if mixed_qkv.dim() != 2:
        raise ValueError("mixed_qkv must be 2-D [N, 2*H*K + HV*V]")
    if final_state.dim() != 4:
        raise ValueError(f"final_state must be 4-D [B, HV, V, K], got {tuple(final_state.shape)}")
    N, width = mixed_qkv.shape
    B, HV, V, K = final_state.shape
    if K != V or K not in HEAD_DIMS:
        raise ValueError(f"heads must be square with a width of {HEAD_DIMS}, got V = {V}, K = {K}")
    qk_dim = width - HV * V
    H = qk_dim // (2 * K)
    if H <= 0 or HV % H != 0 or 2 * H * K != qk_dim:
        raise ValueError(f"cannot infer H from mixed_qkv width {width}")
    args = _lib.PrefillArgs()
    if query_start is None:
        if B == 0 or N % B:
            if N:
                raise ValueError(f"{N} rows are not the same number for each of {B} requests: give query_start")
        args.max_query = N // B if B else 0
        if max_query_len is not None and int(max_query_len) != args.max_query:
            raise ValueError(f"max_query_len is {max_query_len} but every request has {args.max_query} rows")
    else:
        if max_query_len is None or int(max_query_len) < 0:
            raise ValueError("query_start needs max_query_len, the largest number of rows of a request")
        if query_start.dtype != torch.int32 or not query_start.is_contiguous() or tuple(query_start.shape) != (B + 1,):
            raise ValueError(f"query_start must be a contiguous int32 [{B + 1}]")
        args.max_query = min(int(max_query_len), N)
        args.query_start = query_start.data_ptr()
    args.qkv_dtype = _lib.dtype_id(mixed_qkv)
    args.B, args.N, args.H, args.HV, args.K, args.V = B, N, H, HV, K, V
    return args


def _prefill_args(mixed_qkv, a, b, A_log, dt_bias, scale, out, final_state, initial_state, query_start, max_query_len,
                  use_qk_l2norm_in_kernel, status):
    """Checks of a call and the filled argument block."""
    args = _prefill_sizes(mixed_qkv, final_state, query_start, max_query_len)
    N, (B, HV, V, K) = mixed_qkv.shape[0], final_state.shape
    if mixed_qkv.stride(-1) != 1:
        raise ValueError("mixed_qkv must be contiguous in its last dimension")
    _state(final_state, (B, HV, V, K), "final_state")
    if B > 1 and final_state.stride(0) < HV * V * K:
        raise ValueError("final_state: requests' states must not share memory")
    if initial_state is not None:
        _state(initial_state, (B, HV, V, K), "initial_state")
    _lib.need_shape(a, (N, HV), "a")
    _lib.need_shape(b, (N, HV), "b")
    if a.stride(-1) != 1 or b.stride(-1) != 1 or a.dtype != b.dtype:
        raise ValueError("a and b must share a dtype and be contiguous in their last dimension")
    _lib.need_shape(A_log, (HV,), "A_log")
    _lib.need_shape(dt_bias, (HV,), "dt_bias")
    if not A_log.is_contiguous() or not dt_bias.is_contiguous():
        raise ValueError("A_log and dt_bias must be contiguous")
    _lib.need_shape(out, (N, HV, V), "out")
    if out.stride()[1:] != (V, 1):
        raise ValueError("out must be dense within a token (only the token stride may vary)")
    if N > 1 and out.stride(0) < HV * V:
        raise ValueError("out: tokens' rows must not share memory")
    dev = final_state.device
    _lib.same_device(dev, mixed_qkv=mixed_qkv, a=a, b=b, A_log=A_log, dt_bias=dt_bias, out=out, initial_state=initial_state,
                     query_start=query_start)
    args.mixed_qkv, args.stride_mixed_tok = mixed_qkv.data_ptr(), mixed_qkv.stride(0)
    args.a, args.stride_a_tok, args.b, args.stride_b_tok = a.data_ptr(), a.stride(0), b.data_ptr(), b.stride(0)
    args.ab_dtype = _lib.dtype_id(a)
    args.A_log, args.A_log_dtype = A_log.data_ptr(), _lib.dtype_id(A_log)
    args.dt_bias, args.dt_bias_dtype = dt_bias.data_ptr(), _lib.dtype_id(dt_bias)
    if initial_state is not None:
        args.initial_state, args.stride_initial_req = initial_state.data_ptr(), initial_state.stride(0)
    args.final_state, args.stride_final_req = final_state.data_ptr(), final_state.stride(0)
    args.out, args.stride_out_tok, args.out_dtype = out.data_ptr(), out.stride(0), _lib.dtype_id(out)
    args.status = _lib.status_ptr(status, dev)
    args.scale, args.use_qk_l2norm = float(scale), int(bool(use_qk_l2norm_in_kernel))
    return args


def gated_delta_rule_packed_prefill(mixed_qkv, a, b, A_log, dt_bias, scale, out, final_state, initial_state=None, query_start=None,
                                    max_query_len=None, use_qk_l2norm_in_kernel=False, workspace=None, status=None):
    """Every token of every request through the recurrence; fills and returns ``out`` and ``final_state``.

    ``mixed_qkv [N, 2*H*K + HV*V]`` = q | k | v (fp32, bf16 or fp16), ``a, b [N, HV]``, ``A_log, dt_bias [HV]`` and
    ``scale`` as in ``quantized_gated_delta_rule_packed_decode``; ``out [N, HV, V]``; ``initial_state`` (``None`` for zeros)
    and ``final_state`` fp32 ``[B, HV, V, K]``, which may be one tensor.  Every request has ``N / B`` rows, or, with ``query_start [B + 1]``
    (int32), rows ``query_start[b] .. query_start[b + 1] - 1``, ``max_query_len`` of them at most; a request without rows hands its
    state on.  ``query_start`` does not fall: where it does, that is flagged, and what the call's rows and states get is not defined.
    ``K = V`` is 64 or 128.  What is written shares no memory with another part of it or, ``initial_state`` apart, with an input.

    A key that is not finite, and a decay or write strength that is NaN, leave the state of the heads that read them not finite from their token
    on, a value its row of the state, a number of ``initial_state`` its row; outputs ahead of it are what they were.  With
    ``use_qk_l2norm_in_kernel`` the squares of a key's numbers, and of a query's, have to add up to less than fp32's largest number; without it
    products of two keys, and of a key and a query, that are less than 64 tokens apart have to be in its range.

    Few tokens go one by one, more in chunks (the rule is by ``max_query_len``, the type and the number of heads).  The two ways agree within the
    precision of each, not to the bit: in bf16 some two of a thousand outputs fall to the neighbouring number.

    ``workspace`` (uint8, at least :func:`prefill_workspace_bytes`) is allocated by the call when it is not given; calls that may run at the
    same time need one each.  ``status`` as in
    ``quantized_packed_decode``: rows beyond ``max_query_len`` or outside of ``mixed_qkv`` are skipped and flagged
    (``STATUS_BAD_RANGE``)."""
    lib = _lib._lib or _lib.load_library()
    if lib.native.prefill(lib.native_table, mixed_qkv, a, b, A_log, dt_bias, scale, out, final_state, initial_state, query_start,
                          max_query_len, use_qk_l2norm_in_kernel, workspace, status):
        return out, final_state
    # not a call the native path takes as it stands: the checks below say what is wrong with it, if anything
    args = _prefill_args(mixed_qkv, a, b, A_log, dt_bias, scale, out, final_state, initial_state, query_start, max_query_len,
                         use_qk_l2norm_in_kernel, status)
    dev = final_state.device
    _lib.require_cuda(final_state, "final_state")
    with torch.cuda.device(dev):
        need = lib.carry_gdn_prefill_workspace(args)
        _lib.check(min(need, 0), "carry_gdn_prefill_workspace")
        if workspace is None:
            workspace = torch.empty(need, dtype=torch.uint8, device=dev) if need else None
        else:
            _lib.same_device(dev, workspace=workspace)
            if not workspace.is_contiguous() or workspace.numel() * workspace.element_size() < need or workspace.data_ptr() % 16:
                raise ValueError(f"workspace must be contiguous, 16-byte aligned and hold {need} bytes")
        if workspace is not None:
            args.workspace, args.workspace_bytes = workspace.data_ptr(), workspace.numel() * workspace.element_size()
        rc = lib.carry_gdn_prefill(args, _lib.current_stream_ptr(dev))
    _lib.check(rc, "carry_gdn_prefill")
    return out, final_state


def prefill_workspace_bytes(mixed_qkv, final_state, query_start=None, max_query_len=None) -> int:
    """Bytes of workspace that :func:`gated_delta_rule_packed_prefill` needs for a call of these sizes on the state's device (on the
    current one, where the state is on none).  Nothing is read or allocated: tensors of no memory (``device="meta"``) will do."""
    lib = _lib._lib or _lib.load_library()
    args = _prefill_sizes(mixed_qkv, final_state, query_start, max_query_len)
    with torch.cuda.device_of(final_state):
        need = lib.carry_gdn_prefill_workspace(args)
    _lib.check(min(need, 0), "carry_gdn_prefill_workspace")
    return need
