"""8-bit key/value cache of a hybrid model's full-attention layers: append and attention.

A model that mixes Gated-DeltaNet layers with full attention serves from two kinds of per-request memory: the
recurrent state (``quantized_packed_decode``) and, for the attention layers, keys and values that grow with the
context.  This is the second kind, held in 8 bits too:

* a *cache* is the 4-tuple ``(k_codes, k_scale, v_codes, v_scale)`` that :func:`init_quantized_kv` returns: e4m3
  codes ``[pages, HKV, page, D]`` and one fp32 scale for every block of tokens of a head, ``[pages, HKV,
  page // block]`` (the block size is read off the shape); a value is ``code * scale``;
* request ``b`` holds ``lengths[b]`` tokens, token ``j`` of it in page ``block_table[b, j // page]``; a page id ``<= 0``
  (:data:`NULL_BLOCK_ID`) is padding;
* the call's own rows are ``[N, heads, D]``, the same number for every request, or, with ``query_start [B + 1]``, rows
  ``query_start[b] .. query_start[b + 1] - 1`` for request ``b`` (``max_query_len`` bounds them).  ``lengths`` counts
  them: row ``i`` of ``n`` stands at position ``lengths[b] - n + i``.

:func:`quantized_kv_append` writes new tokens, :func:`quantized_paged_attention` attends over what is cached: one
token a request (decode), a few (speculation), a chunk of a prompt.  Scales are powers of two, so that a block whose
scale grows while it fills keeps the codes of its earlier tokens exactly (down to e4m3's subnormals); a speculated token
that is rejected is overwritten by the next append, its scale stays.  (A cache that was filled elsewhere may have any scales from
2^-100 to 2^119, or 0 for blocks whose codes are all 0.)

The calls read nothing back to the host, never synchronise and can be captured in a CUDA graph.  ``status``: as in
``quantized_packed_decode``; ids, lengths and query ranges outside of the call's bounds are skipped and flagged there
(``STATUS_BAD_RANGE``).  There is no CPU path.
"""

from __future__ import annotations

import torch

from .. import _lib
from .quantized_packed_decode import NULL_BLOCK_ID  # noqa: F401

CODES = torch.float8_e4m3fn
HEAD_DIMS = (64, 128)
MAX_BLOCK = 128


def init_quantized_kv(num_pages: int, HKV: int, page: int, D: int, device, block: int = 32):
    """Allocate the cache of one layer, empty: ``(k_codes, k_scale, v_codes, v_scale)``.  Page 0 is the padding page."""
    if D not in HEAD_DIMS:
        raise ValueError(f"head width must be one of {HEAD_DIMS}, got {D}")
    if page <= 0 or block <= 0 or page % 16 or block % 16 or page % block or block > MAX_BLOCK:
        raise ValueError(f"page and block must be multiples of 16, block a divisor of page and at most {MAX_BLOCK}, "
                         f"got page {page}, block {block}")
    codes, scales = (num_pages, HKV, page, D), (num_pages, HKV, page // block)
    return (torch.zeros(codes, dtype=CODES, device=device), torch.zeros(scales, dtype=torch.float32, device=device),
            torch.zeros(codes, dtype=CODES, device=device), torch.zeros(scales, dtype=torch.float32, device=device))


def kv_bytes_per_token(HKV: int, D: int, block: int = 32) -> float:
    """Bytes of cache per token of one layer, scales included."""
    return 2.0 * HKV * (D + 4.0 / block)


def _rows(c, r, rows, lengths, query_start, max_query_len, name, device):
    """Fills ``CarryGdnKvRows`` and the lengths' address from the call's rows ``[N, heads, D]``."""
    if rows.dim() != 3 or rows.stride(-1) != 1:
        raise ValueError(f"{name} must be 3-D [N, heads, D] and contiguous in its last dimension")
    if lengths.dim() != 1 or lengths.dtype != torch.int32 or not lengths.is_contiguous():
        raise ValueError("lengths must be a contiguous int32 [B]")
    r.B, r.N = lengths.shape[0], rows.shape[0]
    if query_start is None:
        if r.B == 0 or r.N % r.B:
            if r.N:
                raise ValueError(f"{r.N} rows of {name} are not the same number for each of {r.B} requests: give query_start")
        r.max_query = r.N // r.B if r.B else 0
        if max_query_len is not None and int(max_query_len) != r.max_query:
            raise ValueError(f"max_query_len is {max_query_len} but every request has {r.max_query} rows")
    else:
        if max_query_len is None or int(max_query_len) < 0:
            raise ValueError("query_start needs max_query_len, the largest number of rows of a request")
        if query_start.dtype != torch.int32 or not query_start.is_contiguous() or tuple(query_start.shape) != (r.B + 1,):
            raise ValueError(f"query_start must be a contiguous int32 [{r.B + 1}]")
        r.max_query = min(int(max_query_len), r.N)
        r.query_start = query_start.data_ptr()
    _lib.same_device(device, lengths=lengths, query_start=query_start, **{name: rows})
    c.lengths = lengths.data_ptr()


def _cache(c, k_codes, k_scale, v_codes, v_scale, block_table, B):
    """Checks of the cache's tensors and the filled ``CarryGdnKvCache``."""
    if k_codes.dim() != 4 or k_codes.dtype != CODES or v_codes.dtype != CODES:
        raise ValueError("k_codes and v_codes must be float8_e4m3fn [pages, HKV, page, D]")
    pages, HKV, page, D = k_codes.shape
    if D not in HEAD_DIMS:
        raise ValueError(f"head width must be one of {HEAD_DIMS}, got {D}")
    if k_scale.dim() != 3 or k_scale.shape[2] == 0 or page % k_scale.shape[2]:
        raise ValueError(f"k_scale must be [pages, HKV, page // block], got {tuple(k_scale.shape)} for pages of {page}")
    per = k_scale.shape[2]
    block = page // per
    if page % 16 or block % 16 or block > MAX_BLOCK:
        raise ValueError(f"page and block must be multiples of 16, block at most {MAX_BLOCK}: got page {page}, block {block}")
    _lib.need_shape(v_codes, (pages, HKV, page, D), "v_codes")
    for name, t in (("k_scale", k_scale), ("v_scale", v_scale)):
        _lib.need_shape(t, (pages, HKV, per), name)
        if t.dtype != torch.float32 or t.stride()[1:] != (per, 1):
            raise ValueError(f"{name} must be fp32 and dense within a page")
    for name, t in (("k_codes", k_codes), ("v_codes", v_codes)):
        if t.stride()[1:] != (page * D, D, 1):
            raise ValueError(f"{name} must be dense within a page (only the page stride may vary)")
        if t.data_ptr() % 16 or t.stride(0) % 16:
            raise ValueError(f"{name}: every page must start on a 16-byte boundary")
    if block_table.dim() != 2 or block_table.dtype != torch.int32 or block_table.shape[0] != B:
        raise ValueError(f"block_table must be int32 [{B}, pages of a request]")
    if block_table.shape[1] > 1 and block_table.stride(1) != 1:
        raise ValueError("block_table must be contiguous in its last dimension")
    _lib.same_device(k_codes.device, k_scale=k_scale, v_codes=v_codes, v_scale=v_scale, block_table=block_table)
    c.k_codes, c.k_scale, c.v_codes, c.v_scale = (t.data_ptr() for t in (k_codes, k_scale, v_codes, v_scale))
    c.stride_k_page, c.stride_ks_page = k_codes.stride(0), k_scale.stride(0)
    c.stride_v_page, c.stride_vs_page = v_codes.stride(0), v_scale.stride(0)
    c.block_table, c.stride_table, c.max_pages = block_table.data_ptr(), block_table.stride(0), block_table.shape[1]
    c.num_pages, c.HKV, c.page, c.block, c.D = pages, HKV, page, block, D


def quantized_kv_append(k, v, k_codes, k_scale, v_codes, v_scale, block_table, lengths, query_start=None,
                        max_query_len=None, status=None):
    """Write the new tokens' keys and values ``k, v [N, HKV, D]`` (fp32, bf16 or fp16) into the cache, in place.

    ``lengths [B]`` already counts the new tokens.  A block whose first token is among them is started afresh; in a
    block with earlier tokens the scale only grows.  A token with a number that is not finite gets a NaN key: the
    queries that see it become NaN, and no others.  Two requests must not append to one page."""
    lib = _lib._lib or _lib.load_library()
    if lib.native.kv_append(lib.native_table, k, v, k_codes, k_scale, v_codes, v_scale, block_table, lengths, query_start,
                            max_query_len, status):
        return
    # not a call the native path takes as it stands: the checks below say what is wrong with it, if anything
    args = _lib.KvAppendArgs()
    dev = k_codes.device
    _rows(args.cache, args.rows, k, lengths, query_start, max_query_len, "k", dev)
    _cache(args.cache, k_codes, k_scale, v_codes, v_scale, block_table, args.rows.B)
    want = (args.rows.N, args.cache.HKV, args.cache.D)
    _lib.need_shape(k, want, "k")
    _lib.need_shape(v, want, "v")
    if v.dtype != k.dtype or v.stride(-1) != 1:
        raise ValueError("k and v must share a dtype and be contiguous in their last dimension")
    _lib.same_device(dev, v=v)
    args.k, args.stride_k_tok, args.stride_k_head = k.data_ptr(), k.stride(0), k.stride(1)
    args.v, args.stride_v_tok, args.stride_v_head = v.data_ptr(), v.stride(0), v.stride(1)
    args.dtype = _lib.dtype_id(k)
    args.status = _lib.status_ptr(status, dev)
    _lib.require_cuda(k_codes, "k_codes")
    with torch.cuda.device(dev):
        rc = lib.carry_gdn_kv_append(args, _lib.current_stream_ptr(dev))
    _lib.check(rc, "carry_gdn_kv_append")


def _attention_args(q, scale, k_codes, k_scale, v_codes, v_scale, out, block_table, lengths, query_start, max_query_len,
                    status):
    args = _lib.KvAttentionArgs()
    dev = k_codes.device
    _rows(args.cache, args.rows, q, lengths, query_start, max_query_len, "q", dev)
    _cache(args.cache, k_codes, k_scale, v_codes, v_scale, block_table, args.rows.B)
    HQ, HKV, D = q.shape[1], args.cache.HKV, args.cache.D
    if HQ == 0 or HQ % HKV:
        raise ValueError(f"{HQ} query heads are not a multiple of {HKV} key/value heads")
    _lib.need_shape(q, (args.rows.N, HQ, D), "q")
    _lib.need_shape(out, (args.rows.N, HQ, D), "out")
    if out.dtype != q.dtype or out.stride(-1) != 1:
        raise ValueError("out must have q's dtype and be contiguous in its last dimension")
    _lib.same_device(dev, out=out)
    args.q, args.stride_q_tok, args.stride_q_head = q.data_ptr(), q.stride(0), q.stride(1)
    args.out, args.stride_out_tok, args.stride_out_head = out.data_ptr(), out.stride(0), out.stride(1)
    args.scale, args.HQ, args.dtype = float(scale), HQ, _lib.dtype_id(q)
    args.status = _lib.status_ptr(status, dev)
    return args


def quantized_paged_attention(q, scale, k_codes, k_scale, v_codes, v_scale, out, block_table, lengths, query_start=None,
                              max_query_len=None, workspace=None, status=None):
    """Causal attention of the rows' queries ``q [N, HQ, D]`` over the cache, into ``out`` (q's shape and dtype);
    returns ``out``.

    ``scale`` multiplies the scores.  Query head ``h`` reads key/value head ``h // (HQ // HKV)``.  A row that sees no
    token (a request of length 0, a padding page) is zero.  ``workspace`` (uint8, at least
    :func:`attention_workspace_bytes`) is allocated by the call when it is not given."""
    lib = _lib._lib or _lib.load_library()
    if lib.native.kv_attention(lib.native_table, q, scale, k_codes, k_scale, v_codes, v_scale, out, block_table, lengths,
                               query_start, max_query_len, workspace, status):
        return out
    args = _attention_args(q, scale, k_codes, k_scale, v_codes, v_scale, out, block_table, lengths, query_start,
                           max_query_len, status)
    dev = k_codes.device
    _lib.require_cuda(k_codes, "k_codes")
    with torch.cuda.device(dev):
        need = lib.carry_gdn_kv_attention_workspace(args)
        _lib.check(min(need, 0), "carry_gdn_kv_attention_workspace")
        if workspace is None:
            workspace = torch.empty(need, dtype=torch.uint8, device=dev) if need else None
        else:
            _lib.same_device(dev, workspace=workspace)
            if not workspace.is_contiguous() or workspace.numel() * workspace.element_size() < need or workspace.data_ptr() % 16:
                raise ValueError(f"workspace must be contiguous, 16-byte aligned and hold {need} bytes")
        if workspace is not None:
            args.workspace, args.workspace_bytes = workspace.data_ptr(), workspace.numel() * workspace.element_size()
        rc = lib.carry_gdn_kv_attention(args, _lib.current_stream_ptr(dev))
    _lib.check(rc, "carry_gdn_kv_attention")
    return out


def attention_workspace_bytes(q, k_codes, k_scale, block_table, query_start=None, max_query_len=None) -> int:
    """Bytes of workspace that :func:`quantized_paged_attention` needs for a call of these sizes on the cache's device
    (on the current one, where the cache is on none)."""
    lib = _lib._lib or _lib.load_library()
    B = block_table.shape[0]
    lengths = torch.empty(B, dtype=torch.int32, device=k_codes.device)
    args = _attention_args(q, 1.0, k_codes, k_scale, k_codes, k_scale, q, block_table, lengths, query_start, max_query_len,
                           None)
    with torch.cuda.device_of(k_codes):
        need = lib.carry_gdn_kv_attention_workspace(args)
    _lib.check(min(need, 0), "carry_gdn_kv_attention_workspace")
    return need
