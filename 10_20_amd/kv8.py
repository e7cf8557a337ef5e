"""K / V cache in 8 bits and its decode attention: pages of 64 tokens of OCP
e4m3fn codes with one fp32 scale for each page and KV head, half the bytes of the
bf16 pools that attention.attend_slots reads.

Pools: k_pool, v_pool [pages, 64, kv_heads, 128] float8_e4m3fn (16-byte aligned, any
strides in multiples of 16, the last dimension contiguous: token-major and
head-major pages alike), k_scale,
v_scale [pages, kv_heads] fp32.  Position i of a request lies in page
table[i // 64], the layout of the page manager.  `store` appends tokens, `attend`
reads them for one query position per row: the first positions of a context or
the Top-K's ids.

Sums are fp32, undivided until the end, and may carry 2^16 times the keys' number
times a value: they are kept for magnitudes between 2^-100 and 2^100.

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


def _bad_pool(name):
    raise ValueError(f"{name} must be float8_e4m3fn [pages, {PAGE}, kv_heads, {DIM}] with a contiguous last dimension")


# (each property of a tensor is asked for once: 0.1-0.3 us of a call whose kernels
# may take 10)
def _pools(k_pool, v_pool, k_scale, v_scale):
    """Pages, KV heads, and the pointers and strides of the pools and scales."""
    shape, kp, vp, ks, vs = k_pool.shape, k_pool.stride(), v_pool.stride(), k_scale.stride(), v_scale.stride()
    if len(shape) != 4 or k_pool.dtype != _E4M3 or kp[3] != 1:
        _bad_pool("k_pool")
    pages, page, heads, dim = shape
    if page != PAGE or dim != DIM or not heads:
        _bad_pool("k_pool")
    if v_pool.shape != shape:
        raise ValueError("k_pool and v_pool must agree")
    if v_pool.dtype != _E4M3 or vp[3] != 1:
        _bad_pool("v_pool")
    each = (pages, heads)
    if k_scale.dtype != _F32 or k_scale.shape != each or (ks[1] != 1 and heads > 1):
        raise ValueError("k_scale must be float32 [pages, kv_heads] with unit inner stride")
    if v_scale.dtype != _F32 or v_scale.shape != each or (vs[1] != 1 and heads > 1):
        raise ValueError("v_scale must be float32 [pages, kv_heads] with unit inner stride")
    return pages, heads, (k_pool.data_ptr(), kp[0], kp[1], kp[2], v_pool.data_ptr(), vp[0], vp[1], vp[2],
                          k_scale.data_ptr(), ks[0], v_scale.data_ptr(), vs[0], pages)


def _vector(name, t, n):
    if t.dtype != _I32 or t.shape != (n,) or not t.is_contiguous():
        raise ValueError(f"{name} must be a contiguous int32 [{n}] tensor")


# (sizes alone decide: asked of the library once for each)
@functools.lru_cache(maxsize=4096)
def _workspace_bytes(index, *sizes):
    return _lib.workspace_bytes("v1_kv8_attend_workspace", index, *sizes)


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
    pages, heads, pools = _pools(k_pool, v_pool, k_scale, v_scale)
    shape, ks, vs = k.shape, k.stride(), v.stride()
    tokens = shape[0] if len(shape) == 3 else -1
    if shape != (tokens, heads, DIM) or k.dtype != _BF16 or ks[2] != 1:
        raise ValueError(f"k must be bfloat16 [tokens, {heads}, {DIM}] with a contiguous last dimension")
    if v.shape != shape:
        raise ValueError("k and v must be of one shape")
    if v.dtype != _BF16 or vs[2] != 1:
        raise ValueError(f"v must be bfloat16 [tokens, {heads}, {DIM}] with a contiguous last dimension")
    ts = table.stride()
    if table.dtype != _I32 or len(ts) != 2 or (ts[1] != 1 and table.shape[1]):
        raise ValueError("table must be int32 [requests, entries] with unit inner stride")
    requests, entries = table.shape
    _vector("starts", starts, requests)
    _vector("cu_tokens", cu_tokens, requests + 1)
    _lib.call_packed("v1_kv8_store", k, k.data_ptr(), ks[0], ks[1], v.data_ptr(), vs[0], vs[1], *pools,
                     table.data_ptr(), ts[0], starts.data_ptr(), cu_tokens.data_ptr(), entries, tokens, requests, heads)


def attend(q, k_pool, v_pool, k_scale, v_scale, table, lens=None, ids=None, softmax_scale=None, out=None, return_lse=False):
    """out[r, h] = sum_j softmax_j(scale * q[r, h] . k_j) v_j over the keys of row r,
    query head h reading KV head h // (heads / kv_heads) (at most 16 heads a KV head).

    q:     [rows, heads, 128] bf16
    table: [rows, entries] int32 pages of each row's positions, or [entries] for all
    ids:   [rows, keys] int32 positions, or None: positions 0, 1, ...
    lens:  [rows] int32: the first lens[r] entries of ids (or positions) are row r's;
           None: all

    Ids below zero, past the table or in pages outside the pool are not attended.  A
    row without keys gives zeros and -inf, one whose keys all score -inf NaN and
    -inf.  softmax_scale > 0, default 1 / sqrt(128).
    Returns out [rows, heads, 128] bf16, and with return_lse the natural log of the
    sum of exponentials, [rows, heads] fp32."""
    _lib.require_gpu(q, k_pool, v_pool, k_scale, v_scale, table, lens, ids, out)
    pages, kv_heads, pools = _pools(k_pool, v_pool, k_scale, v_scale)
    shape, qs = q.shape, q.stride()
    if len(shape) != 3 or shape[2] != DIM or q.dtype != _BF16 or qs[2] != 1:
        raise ValueError(f"q must be bfloat16 [rows, heads, {DIM}] with a contiguous last dimension")
    rows, heads, _ = shape
    group = heads // kv_heads
    if not heads or heads % kv_heads or group > 16:
        raise ValueError("query heads must be a multiple of KV heads, at most 16 per KV head")
    of, ts = table.shape, table.stride()
    dims = len(of)
    if table.dtype != _I32 or not (dims == 1 or (dims == 2 and of[0] == rows)):
        raise ValueError("table must be int32 [entries] or [rows, entries]")
    entries = of[-1]
    if entries and ts[-1] != 1:
        raise ValueError("table must have unit inner stride")
    ids_ptr = ids_stride = lens_ptr = 0
    if ids is not None:
        of, at = ids.shape, ids.stride()
        if ids.dtype != _I32 or len(of) != 2 or of[0] != rows or (at[1] != 1 and of[1]):
            raise ValueError("ids must be int32 [rows, keys] with unit inner stride")
        keys, ids_ptr, ids_stride = of[1], ids.data_ptr(), at[0]
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
    o_row, o_head, o_dim = out.stride() if out.dim() == 3 else (0, 0, 0)
    if o_dim != 1 or out.dtype != _BF16 or out.shape != shape:
        raise ValueError(f"out must be bfloat16 [{rows}, {heads}, {DIM}] with a contiguous last dimension")
    lse = q.new_empty((rows, heads), dtype=_F32) if return_lse else None
    # (the sums of a row's parts are the call's own, as in attention.attend_slots)
    ws_bytes = _workspace_bytes(q.get_device(), rows, kv_heads, group, keys, lens is not None)
    ws = q.new_empty((ws_bytes,), dtype=torch.uint8) if ws_bytes else None
    _lib.call_packed("v1_kv8_attend", q, q.data_ptr(), qs[0], qs[1], *pools, table.data_ptr(), ts[0] if dims == 2 else 0,
                     ids_ptr, ids_stride, lens_ptr, out.data_ptr(), o_row, o_head, _lib.ptr(lse), _lib.ptr(ws), ws_bytes,
                     entries, rows, kv_heads, group, keys, scale)
    return (out, lse) if return_lse else out
