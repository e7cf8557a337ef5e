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
import functools
import math

import torch

from . import _lib

PAGE, DIM = 64, 128


_DEFAULT_SCALE = 1.0 / math.sqrt(DIM)
_BF16, _I32, _F32, _E4M3 = torch.bfloat16, torch.int32, torch.float32, torch.float8_e4m3fn


def _pools(k_pool, v_pool, k_scale, v_scale):
    shape = k_pool.shape
    if len(shape) != 4 or shape[1] != PAGE or shape[3] != DIM or not shape[2]:
        raise ValueError(f"k_pool must be float8_e4m3fn [pages, {PAGE}, kv_heads, {DIM}] with a contiguous last dimension")
    if v_pool.shape != shape:
        raise ValueError("k_pool and v_pool must agree")
    for name, t in (("k_pool", k_pool), ("v_pool", v_pool)):
        if t.dtype != _E4M3 or t.stride(3) != 1:
            raise ValueError(f"{name} must be float8_e4m3fn [pages, {PAGE}, kv_heads, {DIM}] with a contiguous last dimension")
    pages, _, heads, _ = shape
    for name, t in (("k_scale", k_scale), ("v_scale", v_scale)):
        if t.dtype != _F32 or t.shape != (pages, heads) or (heads > 1 and t.stride(1) != 1):
            raise ValueError(f"{name} must be float32 [pages, kv_heads] with unit inner stride")
    return pages, heads


def _vector(name, t, n):
    if t.dtype != _I32 or t.shape != (n,) or not t.is_contiguous():
        raise ValueError(f"{name} must be a contiguous int32 [{n}] tensor")


# (sizes alone decide: asked of the library once for each)
@functools.lru_cache(maxsize=4096)
def _workspace_bytes(index, *sizes):
    with torch.cuda.device(index):
        return _lib.lib().v1_kv8_attend_workspace(*sizes)


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
        if t.dtype != _BF16 or t.dim() != 3 or t.shape[1:] != (heads, DIM) or t.stride(2) != 1:
            raise ValueError(f"{name} must be bfloat16 [tokens, {heads}, {DIM}] with a contiguous last dimension")
    tokens = k.shape[0]
    if v.shape[0] != tokens:
        raise ValueError("k and v must be of one shape")
    if table.dtype != _I32 or table.dim() != 2 or (table.shape[1] and table.stride(1) != 1):
        raise ValueError("table must be int32 [requests, entries] with unit inner stride")
    requests, entries = table.shape
    _vector("starts", starts, requests)
    _vector("cu_tokens", cu_tokens, requests + 1)
    _lib.call_packed("v1_kv8_store", k, k.data_ptr(), *k.stride()[:2], v.data_ptr(), *v.stride()[:2],
                     k_pool.data_ptr(), *k_pool.stride()[:3], v_pool.data_ptr(), *v_pool.stride()[:3], k_scale.data_ptr(),
                     k_scale.stride(0), v_scale.data_ptr(), v_scale.stride(0), pages, table.data_ptr(), table.stride(0),
                     starts.data_ptr(), cu_tokens.data_ptr(), entries, tokens, requests, heads)


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
    if q.dim() != 3 or q.shape[2] != DIM or q.dtype != _BF16 or q.stride(2) != 1:
        raise ValueError(f"q must be bfloat16 [rows, heads, {DIM}] with a contiguous last dimension")
    rows, heads, _ = q.shape
    group = heads // kv_heads
    if not heads or heads % kv_heads or group > 16:
        raise ValueError("query heads must be a multiple of KV heads, at most 16 per KV head")
    dims, entries = table.dim(), table.shape[-1]
    if table.dtype != _I32 or not (dims == 1 or (dims == 2 and table.shape[0] == rows)):
        raise ValueError("table must be int32 [entries] or [rows, entries]")
    if entries and table.stride(-1) != 1:
        raise ValueError("table must have unit inner stride")
    ids_ptr = ids_stride = lens_ptr = 0
    if ids is not None:
        if ids.dtype != _I32 or ids.dim() != 2 or ids.shape[0] != rows or (ids.shape[1] and ids.stride(1) != 1):
            raise ValueError("ids must be int32 [rows, keys] with unit inner stride")
        keys, ids_ptr, ids_stride = ids.shape[1], ids.data_ptr(), ids.stride(0)
    else:
        keys = entries * PAGE
        if keys >= 1 << 31:
            raise ValueError("positions must stay below 2**31")
    if lens is not None:
        _vector("lens", lens, rows)
        lens_ptr = lens.data_ptr()
    scale = _DEFAULT_SCALE if softmax_scale is None else float(softmax_scale)
    if not 0.0 < scale < math.inf:
        raise ValueError("softmax_scale must be positive and finite")
    if pages == 0 or entries == 0:
        keys = 0
    if out is None:
        out = q.new_empty((rows, heads, DIM))
    elif out.dtype != _BF16 or out.shape != (rows, heads, DIM) or out.stride(2) != 1:
        raise ValueError(f"out must be bfloat16 [{rows}, {heads}, {DIM}] with a contiguous last dimension")
    lse = q.new_empty((rows, heads), dtype=_F32) if return_lse else None
    # (the sums of a row's parts are the call's own, as in attention.attend_slots)
    ws_bytes = _workspace_bytes(q.get_device(), rows, kv_heads, group, keys, lens is not None)
    ws = q.new_empty((ws_bytes,), dtype=torch.uint8) if ws_bytes else None
    _lib.call_packed("v1_kv8_attend", q, q.data_ptr(), *q.stride()[:2], k_pool.data_ptr(),
                     *k_pool.stride()[:3], v_pool.data_ptr(), *v_pool.stride()[:3], k_scale.data_ptr(), k_scale.stride(0),
                     v_scale.data_ptr(), v_scale.stride(0), pages, table.data_ptr(), table.stride(0) if dims == 2 else 0,
                     ids_ptr, ids_stride, lens_ptr, out.data_ptr(), *out.stride()[:2], _lib.ptr(lse), _lib.ptr(ws),
                     ws_bytes, entries, rows, kv_heads, group, keys, scale)
    return (out, lse) if return_lse else out
