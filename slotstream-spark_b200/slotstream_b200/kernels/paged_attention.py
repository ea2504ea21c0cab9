"""Attention over a paged key-value cache (additive API): decode steps and ragged prompts.

The reference's attention lies outside the path that this package replaces; these entry points give the layers between
the MoE layers. ``k_pages`` / ``v_pages`` are [pages, kv_heads, page_size, head_dim] (bf16 or fp16, any strides that are
multiples of 8 with the last dimension contiguous, equal for both), e.g. ``PagedKvCache.k(layer)`` / ``v(layer)``;
``page_table`` int32 [rows, max_pages]; ``lengths`` int32 [rows] counts the tokens in the cache, the queries' own among
them. The queries of a sequence are its newest tokens, so query i of q sits at position lengths - q + i; it sees the
tokens t at or before it, and where ``window`` > 0 only those less than ``window`` back, and the first ``sinks``.
A query that sees nothing gives zeros and a log-sum-exp of -inf. ``ids`` (int32) maps batch row b to its table row.

Scores, softmax statistics and sums are fp32; the softmax weights are rounded to the inputs' type for the tensor cores.
``lse`` (fp32, optional output) is the natural log-sum-exp of the scaled scores, for joining with other parts. ``err``
(int32 [1], e.g. ``PagedKvCache.err``) gets error bits; without it nothing tells of a missing page, a bad id or a prompt
whose kernel gave up waiting (rows of ``out`` are then left unwritten), so a program passes it; ``ws`` (uint8,
``workspace_bytes``) avoids the allocation of a workspace, which capture in a CUDA graph with caller-owned memory wants."""
import ctypes
import math

import torch

from .. import _lib

_TYPES = {torch.bfloat16: _lib.BF16, torch.float16: _lib.F16}
_WS = {}


def workspace_bytes(head_dim: int, n: int, rows: int, heads: int, kv_heads: int, page_size: int, max_pages: int,
                    window: int = 0, sinks: int = 0, prefill: bool = False) -> int:
    """Bytes of ``ws`` for ``n`` sequences with ``rows`` query tokens in all (0: none is needed). Small calls need none."""
    key = (head_dim, n, rows, heads, kv_heads, page_size, max_pages, window, sinks, prefill, _lib.device_index())
    got = _WS.get(key)
    if got is None:
        b = ctypes.c_int64()
        if not prefill and n and rows % n:
            raise ValueError(f"{rows} query tokens are no multiple of {n} sequences")
        args = _lib.ATTN_ARGS.pack(*([0] * 18), rows, 0, n, rows // n if n else 0, heads, kv_heads, head_dim, page_size, 0, 0,
                                   max_pages, window, sinks, 1.0)
        _lib.check(_lib.lib().ssb_attn_workspace(args, int(prefill), ctypes.byref(b)), "attention workspace")
        if len(_WS) > 4096:
            _WS.clear()
        got = _WS[key] = b.value
    return got


def _bad_pages(q, k_pages, v_pages, dim, heads):
    """The refusal for the cache's views (built only when one of the checks in the calls below fails)."""
    if q.dtype not in _TYPES or k_pages.dtype != q.dtype or v_pages.dtype != q.dtype:
        return ValueError("q, k_pages and v_pages must all be bf16 or all fp16")
    if k_pages.dim() != 4 or k_pages.shape != v_pages.shape or k_pages.shape[3] != dim:
        return ValueError(f"k_pages and v_pages must both be [pages, kv_heads, page_size, {dim}]")
    if k_pages.stride() != v_pages.stride() or k_pages.stride(3) != 1:
        return ValueError("k_pages and v_pages must have the same strides, the last one 1")
    return ValueError(f"{heads} query heads are no multiple of {k_pages.shape[1]} key heads")


def _attend(call, what, q, heads, dim, n, q_len, tokens, starts, q_strides, k_pages, v_pages, page_table, lengths, out, lse, scale,
            window, sinks, ids, err, ws):
    """The checks, allocations and arguments that both entry points share."""
    tag = _TYPES.get(q.dtype)
    ps, ks = k_pages.shape, k_pages.stride()
    if tag is None or k_pages.dtype != q.dtype or v_pages.dtype != q.dtype or len(ps) != 4 or v_pages.shape != ps \
            or v_pages.stride() != ks or ks[3] != 1 or ps[3] != dim or heads % ps[1]:
        raise _bad_pages(q, k_pages, v_pages, dim, heads)
    if page_table.dtype != torch.int32 or page_table.dim() != 2 or not page_table.is_contiguous():
        raise ValueError("page_table must be a contiguous int32 [rows, max_pages]")
    rows, max_pages = page_table.shape
    if lengths.dtype != torch.int32 or lengths.shape != (rows,) or not lengths.is_contiguous():
        raise ValueError("lengths must be a contiguous int32 vector, one per row of page_table")
    if ids is not None:
        if ids.dtype != torch.int32 or ids.shape != (n,) or not ids.is_contiguous():
            raise ValueError(f"ids must be a contiguous int32 vector of {n}")
    elif n > rows:
        raise ValueError(f"{n} sequences, but page_table has {rows} rows")
    if not (0 <= window < 2 ** 31 and 0 <= sinks < 2 ** 31):
        raise ValueError("window and sinks must not be negative, nor past 32 bits")
    if scale is None:
        scale = dim ** -0.5
    elif not 0 < scale < math.inf:
        raise ValueError("scale must be positive and finite")
    if err is not None and (err.dtype != torch.int32 or err.numel() != 1):
        raise ValueError("err must be one int32")
    shape = q.shape
    if out is None:
        out = torch.empty_like(q, memory_format=torch.contiguous_format)
    elif out.dtype != q.dtype or out.shape != shape or not out.is_contiguous():
        raise ValueError("out must be contiguous, with q's shape and type")
    if lse is not None and (lse.dtype != torch.float32 or lse.shape != shape[:-1] or not lse.is_contiguous()):
        raise ValueError("lse must be a contiguous fp32 tensor of q's shape without the last dimension")
    need = workspace_bytes(dim, n, tokens, heads, ps[1], ps[2], max_pages, window, sinks, starts is not None)
    if ws is None:
        if need:
            ws = torch.empty(need, dtype=torch.uint8, device=q.device)
    elif ws.dtype != torch.uint8 or not ws.is_contiguous() or ws.numel() < need:
        raise ValueError(f"ws must be a contiguous uint8 tensor of at least {need} bytes")
    p = _lib.ptr
    args = _lib.ATTN_ARGS.pack(
        p(q), p(k_pages), p(v_pages), *q_strides, ks[0], ks[1], ks[2], p(page_table), p(lengths), 0 if ids is None else p(ids),
        0 if starts is None else p(starts), p(out), 0 if lse is None else p(lse), 0 if err is None else p(err),
        0 if ws is None else p(ws), need, tokens, tag, n, q_len, heads, ps[1], dim, ps[2], ps[0], rows, max_pages, window, sinks,
        scale)
    rc = call(args, _lib.stream())
    if rc:
        _lib.check(rc, what)
    return out


def attn_decode(q, k_pages, v_pages, page_table, lengths, out=None, *, lse=None, scale=None, window: int = 0,
                sinks: int = 0, ids=None, err=None, ws=None):
    """q [n, q_len, heads, head_dim] -> out of the same shape: the ``q_len`` newest tokens of every sequence (one of a
    decode step, a few of a speculative verify; q_len * heads / kv_heads <= 128). ``scale`` defaults to
    1 / sqrt(head_dim)."""
    qs = q.stride()
    if len(qs) != 4 or qs[3] != 1:
        raise ValueError("q must be [n, q_len, heads, head_dim] with a contiguous head_dim")
    n, q_len, heads, dim = q.shape
    return _attend(_lib.lib().ssb_attn_decode, "attn_decode", q, heads, dim, n, q_len, n * q_len, None, qs[:3], k_pages, v_pages,
                   page_table, lengths, out, lse, scale, window, sinks, ids, err, ws)


def attn_prefill(q, k_pages, v_pages, page_table, lengths, starts, out=None, *, lse=None, scale=None, window: int = 0,
                 sinks: int = 0, ids=None, err=None, ws=None):
    """q [rows, heads, head_dim] -> out of the same shape. Rows ``starts[b]`` to ``starts[b + 1]`` (int32 [n + 1], on the
    device, rising) are the newest tokens of sequence b: whole prompts, or chunks after cached ones. Rows outside
    every sequence are not written."""
    qs = q.stride()
    if len(qs) != 3 or qs[2] != 1:
        raise ValueError("q must be [rows, heads, head_dim] with a contiguous head_dim")
    if starts.dtype != torch.int32 or starts.dim() != 1 or starts.numel() < 1 or not starts.is_contiguous():
        raise ValueError("starts must be a contiguous int32 vector of at least one element")
    total, heads, dim = q.shape
    return _attend(_lib.lib().ssb_attn_prefill, "attn_prefill", q, heads, dim, starts.shape[0] - 1, 0, total, starts, (0, qs[0], qs[1]),
                   k_pages, v_pages, page_table, lengths, out, lse, scale, window, sinks, ids, err, ws)
