"""K / V cache in 8 bits and its decode attention: pages of 64 tokens of OCP
e4m3fn codes with one fp32 scale for each page and KV head, half the bytes of the
bf16 pools that attention.attend_slots reads.

Pools: k_pool, v_pool [pages, 64, kv_heads, 128] float8_e4m3fn (any strides, the
last dimension contiguous: token-major and head-major pages alike), k_scale,
v_scale [pages, kv_heads] fp32.  Position i of a request lies in page
table[i // 64], the layout of the page manager.  `store` appends tokens, `attend`
reads them for one query position per row: the first positions of a context or
the Top-K's ids.

Every call launches on the current stream of its tensors' device, never
synchronises, and raises ValueError for arguments that do not fit.
"""
import math

import torch

from . import _lib

PAGE, DIM = 64, 128


def _pools(k_pool, v_pool, k_scale, v_scale):
    for name, t in (("k_pool", k_pool), ("v_pool", v_pool)):
        if t.dtype != torch.float8_e4m3fn or t.dim() != 4 or t.shape[1] != PAGE or t.shape[3] != DIM or t.stride(3) != 1:
            raise ValueError(f"{name} must be float8_e4m3fn [pages, {PAGE}, kv_heads, {DIM}] with a contiguous last dimension")
    if k_pool.shape != v_pool.shape or not k_pool.shape[2]:
        raise ValueError("k_pool and v_pool must agree and have KV heads")
    pages, heads = k_pool.shape[0], k_pool.shape[2]
    for name, t in (("k_scale", k_scale), ("v_scale", v_scale)):
        if t.dtype != torch.float32 or tuple(t.shape) != (pages, heads) or (heads > 1 and t.stride(1) != 1):
            raise ValueError(f"{name} must be float32 [pages, kv_heads] with unit inner stride")
    return pages, heads


def _strides(t):
    return _lib.ptr(t), t.stride(0), t.stride(1), t.stride(2)


def _vector(name, t, n):
    if t.dtype != torch.int32 or tuple(t.shape) != (n,) or not t.is_contiguous():
        raise ValueError(f"{name} must be a contiguous int32 [{n}] tensor")


def store(k, v, k_pool, v_pool, k_scale, v_scale, table, starts, cu_tokens):
    """Appends to request r the tokens cu_tokens[r] .. cu_tokens[r + 1] - 1 of k and v
    [tokens, kv_heads, 128] bf16, at positions starts[r], starts[r] + 1, ... of its
    row of `table` [requests, entries] int32.

    A page written from its first token gets a scale of its own: the smallest power
    of two s (2^-126 at least) with |x| <= 448 s for the new tokens' finite numbers.
    One that holds older tokens keeps its scale, or takes that one where it is
    larger, and its older codes are then rounded again.  A code is the nearest e4m3
    value of x / s (ties to even); infinities are stored as +-448 s, NaN as NaN.
    Rows of a page behind the last new token stay as they are.  Positions past the
    table, pages outside the pool and requests with a negative start are skipped; a
    page is appended to by one request of a call (pages shared by several are full)."""
    _lib.require_gpu(k, v, k_pool, v_pool, k_scale, v_scale, table, starts, cu_tokens)
    pages, heads = _pools(k_pool, v_pool, k_scale, v_scale)
    for name, t in (("k", k), ("v", v)):
        if t.dtype != torch.bfloat16 or t.dim() != 3 or tuple(t.shape[1:]) != (heads, DIM) or t.stride(2) != 1:
            raise ValueError(f"{name} must be bfloat16 [tokens, {heads}, {DIM}] with a contiguous last dimension")
    if v.shape != k.shape:
        raise ValueError("k and v must be of one shape")
    if table.dtype != torch.int32 or table.dim() != 2 or (table.shape[1] and table.stride(1) != 1):
        raise ValueError("table must be int32 [requests, entries] with unit inner stride")
    requests = table.shape[0]
    _vector("starts", starts, requests)
    _vector("cu_tokens", cu_tokens, requests + 1)
    _lib.call("v1_kv8_store", _lib.ptr(k), k.stride(0), k.stride(1), _lib.ptr(v), v.stride(0), v.stride(1),
              *_strides(k_pool), *_strides(v_pool), _lib.ptr(k_scale), k_scale.stride(0), _lib.ptr(v_scale),
              v_scale.stride(0), pages, _lib.ptr(table), table.stride(0), table.shape[1], _lib.ptr(starts),
              _lib.ptr(cu_tokens), k.shape[0], requests, heads, _lib.stream_of(k))


def attend(q, k_pool, v_pool, k_scale, v_scale, table, lens=None, ids=None, softmax_scale=None, out=None, return_lse=False):
    """out[r, h] = sum_j softmax_j(scale * q[r, h] . k_j) v_j over the keys of row r,
    query head h reading KV head h // (heads / kv_heads) (at most 16 heads a KV head).

    q:     [rows, heads, 128] bf16
    table: [rows, entries] int32 pages of each row's positions, or [entries] for all
    ids:   [rows, keys] int32 positions, or None: positions 0, 1, ...
    lens:  [rows] int32: the first lens[r] entries of ids (or positions) are row r's;
           None: all

    Ids below zero, past the table or in pages outside the pool are not attended.  A
    row without keys gives zeros and -inf.  softmax_scale > 0, default 1 / sqrt(128).
    Returns out [rows, heads, 128] bf16, and with return_lse the natural log of the
    sum of exponentials, [rows, heads] fp32."""
    _lib.require_gpu(q, k_pool, v_pool, k_scale, v_scale, table, lens, ids, out)
    pages, kv_heads = _pools(k_pool, v_pool, k_scale, v_scale)
    if q.dim() != 3 or q.shape[2] != DIM or q.dtype != torch.bfloat16 or q.stride(2) != 1:
        raise ValueError(f"q must be bfloat16 [rows, heads, {DIM}] with a contiguous last dimension")
    rows, heads, _ = q.shape
    if not heads or heads % kv_heads or heads // kv_heads > 16:
        raise ValueError("query heads must be a multiple of KV heads, at most 16 per KV head")
    if table.dtype != torch.int32 or table.dim() not in (1, 2) or (table.dim() == 2 and table.shape[0] != rows):
        raise ValueError("table must be int32 [entries] or [rows, entries]")
    entries = table.shape[-1]
    if entries and table.stride(-1) != 1:
        raise ValueError("table must have unit inner stride")
    if ids is not None:
        if ids.dtype != torch.int32 or ids.dim() != 2 or ids.shape[0] != rows or (ids.shape[1] and ids.stride(1) != 1):
            raise ValueError("ids must be int32 [rows, keys] with unit inner stride")
        keys = ids.shape[1]
    else:
        keys = entries * PAGE
        if keys >= 1 << 31:
            raise ValueError("positions must stay below 2**31")
    if lens is not None:
        _vector("lens", lens, rows)
    scale = float(softmax_scale) if softmax_scale is not None else 1.0 / math.sqrt(DIM)
    if not 0.0 < scale < math.inf:
        raise ValueError("softmax_scale must be positive and finite")
    if pages == 0 or entries == 0:
        keys = 0
    if out is None:
        out = torch.empty((rows, heads, DIM), device=q.device, dtype=torch.bfloat16)
    elif out.dtype != torch.bfloat16 or tuple(out.shape) != (rows, heads, DIM) or out.stride(2) != 1:
        raise ValueError(f"out must be bfloat16 [{rows}, {heads}, {DIM}] with a contiguous last dimension")
    lse = torch.empty((rows, heads), device=q.device, dtype=torch.float32) if return_lse else None
    # (the sums of a row's parts are the call's own, as in attention.attend_slots)
    ws_bytes = _lib.lib().v1_kv8_attend_workspace(rows, kv_heads, heads // kv_heads, keys, lens is not None)
    ws = torch.empty(ws_bytes, device=q.device, dtype=torch.uint8) if ws_bytes else None
    _lib.call("v1_kv8_attend", _lib.ptr(q), q.stride(0), q.stride(1), *_strides(k_pool), *_strides(v_pool),
              _lib.ptr(k_scale), k_scale.stride(0), _lib.ptr(v_scale), v_scale.stride(0), pages, _lib.ptr(table),
              table.stride(0) if table.dim() == 2 else 0, entries, _lib.ptr(ids),
              ids.stride(0) if ids is not None else 0, _lib.ptr(lens), rows, kv_heads, heads // kv_heads, keys, scale,
              _lib.ptr(out), out.stride(0), out.stride(1), _lib.ptr(lse), _lib.ptr(ws), ws_bytes, _lib.stream_of(q))
    return (out, lse) if return_lse else out
