"""K / V cache of 16-bit numbers in pages of 64 tokens, for whole requests: tokens
appended with their keys rotated, attention of prompts, chunks, single tokens and
drafted trees over the pages, and the accepted drafts' rows moved to the end of
their context.  (attention.attend_slots reads slots of the same layout for the
Top-K's ids of single tokens; kv8 holds pages in 8 bits.)

Pools: k_pool, v_pool [pages, 64, kv_heads, 128] bfloat16 or float16 (16-byte
aligned, any strides in multiples of 8, the last dimension contiguous: token-major
and head-major pages alike; `attend` takes tokens of a page less than 2**25 numbers apart).  Position i of a request lies in page table[r, i // 64],
the layout of the page manager.

A step of drafted trees: `append` writes the drafts behind the context, each at the
angle of its depth (`positions`), `attend_tree` lets each see the context and its
ancestors, and `keep` moves the rows of the accepted ones together.

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
MOST_DRAFTS = 256

_DEFAULT_SCALE = 1.0 / math.sqrt(DIM)
_I32, _F32 = torch.int32, torch.float32
_TYPES = (torch.bfloat16, torch.float16)


def _bad_pool(name):
    raise ValueError(f"{name} must be bfloat16 or float16 [pages, {PAGE}, kv_heads, {DIM}] with a contiguous last dimension")


# (each property of a tensor is asked for once: 0.1-0.3 us of a call whose kernels
# may take 5)
def _pools(k_pool, v_pool):
    """Type, pages, KV heads, and the pointers and strides of the pools."""
    shape, kp, vp, dtype = k_pool.shape, k_pool.stride(), v_pool.stride(), k_pool.dtype
    if len(shape) != 4 or dtype not in _TYPES or kp[3] != 1:
        _bad_pool("k_pool")
    pages, page, heads, dim = shape
    if page != PAGE or dim != DIM or not heads:
        _bad_pool("k_pool")
    if v_pool.shape != shape or v_pool.dtype != dtype:
        raise ValueError("k_pool and v_pool must agree")
    if vp[3] != 1:
        _bad_pool("v_pool")
    return dtype, pages, heads, (k_pool.data_ptr(), kp[0], kp[1], kp[2], v_pool.data_ptr(), vp[0], vp[1], vp[2], pages)


def _vector(name, t, n):
    if t.dtype != _I32 or t.shape != (n,) or not t.is_contiguous():
        raise ValueError(f"{name} must be a contiguous int32 [{n}] tensor")


def _table(table):
    ts = table.stride()
    if table.dtype != _I32 or len(ts) != 2 or (ts[1] != 1 and table.shape[1]):
        raise ValueError("table must be int32 [requests, entries] with unit inner stride")
    return (*table.shape, ts[0])


def _rows(name, t, dtype, tokens, heads):
    """Strides of a tensor of `heads` rows of each token (None: any number of either)."""
    shape, s = t.shape, t.stride()
    if len(shape) != 3 or shape[2] != DIM or t.dtype != dtype or s[2] != 1 or (tokens is not None and shape[0] != tokens) or (
            heads is not None and shape[1] != heads):
        raise ValueError(f"{name} must be {str(dtype)[6:]} [{'tokens' if tokens is None else tokens}, "
                         f"{'heads' if heads is None else heads}, {DIM}] with a contiguous last dimension")
    return s


# (sizes alone decide: asked of the library once for each)
@functools.lru_cache(maxsize=4096)
def _workspace_bytes(index, *sizes):
    return _lib.workspace_bytes("v1_paged_attend_workspace", index, *sizes)


def rotations(positions, rotated=DIM, base=10000.0, device=None):
    """The table that `append` takes: cosines, then sines, of the angles i * base ** (-2 p / rotated)
    of positions 0 <= i < `positions` and pairs 0 <= p < rotated / 2, [positions, rotated] fp32
    (angles in 64 bits, rounded once).  A model with other angles builds its own."""
    if rotated <= 0 or rotated > DIM or rotated % 16:
        raise ValueError(f"rotated must be a multiple of 16 up to {DIM}")
    half = rotated // 2
    pairs = torch.arange(half, device=device, dtype=torch.float64)
    angles = torch.arange(positions, device=device, dtype=torch.float64)[:, None] * base ** (-pairs / half)
    return torch.cat([angles.cos(), angles.sin()], 1).float()


def append(q, k, v, k_pool, v_pool, table, starts, cu_tokens, rotations, positions=None, interleaved=False, out=None):
    """Appends to request r the tokens cu_tokens[r] .. cu_tokens[r + 1] - 1 of k and v
    [tokens, kv_heads, 128], at positions starts[r], starts[r] + 1, ... of its row of
    `table` [requests, entries] int32: v as it is, k rotated.  Returns q [tokens,
    heads, 128] rotated alike, in `out` (which may be q) or a new tensor; q None: None.

    rotations: [n, rotated] fp32, cosines then sines of the rotated / 2 pairs (rotated
               a multiple of 16 up to 128; numbers past it are not turned)
    positions: [tokens] int32, the row of `rotations` of each token, or None: its
               position (drafted trees give the context's length plus the depth)
    interleaved: a pair is numbers 2i and 2i + 1; else i and i + rotated / 2

    x, y -> x cos - y sin, y cos + x sin in fp32, rounded once.  Tokens outside the
    requests, or whose row of `rotations` is not there, are skipped: neither stored
    nor written to `out`.  A request that starts below zero is not stored, none of its
    tokens, and positions past the table and pages outside the pool are not written to.
    Two tokens of a call have positions of their own."""
    _lib.require_gpu(q, k, v, k_pool, v_pool, table, starts, cu_tokens, rotations, positions, out)
    dtype, pages, kv_heads, pools = _pools(k_pool, v_pool)
    ks = _rows("k", k, dtype, None, kv_heads)
    tokens = k.shape[0]
    vs = _rows("v", v, dtype, tokens, kv_heads)
    heads, qs, os, q_ptr, o_ptr = 0, (0, 0), (0, 0), 0, 0
    if q is not None:
        qs = _rows("q", q, dtype, tokens, None)
        heads = q.shape[1]
        if out is None:
            out = q.new_empty((tokens, heads, DIM))
        os = _rows("out", out, dtype, tokens, heads)
        q_ptr, o_ptr = q.data_ptr(), out.data_ptr()
    elif out is not None:
        raise ValueError("out without q")
    requests, entries, ts = _table(table)
    _vector("starts", starts, requests)
    _vector("cu_tokens", cu_tokens, requests + 1)
    of, rs = rotations.shape, rotations.stride()
    if rotations.dtype != _F32 or len(of) != 2 or not of[1] or of[1] > DIM or of[1] % 16 or rs[1] != 1:
        raise ValueError(f"rotations must be float32 [positions, rotated], rotated a multiple of 16 up to {DIM}, with unit inner stride")
    at = 0
    if positions is not None:
        _vector("positions", positions, tokens)
        at = positions.data_ptr()
    _lib.call_packed("v1_paged_append", k, q_ptr, qs[0], qs[1], k.data_ptr(), ks[0], ks[1], v.data_ptr(), vs[0], vs[1], o_ptr, os[0],
                     os[1], *pools, table.data_ptr(), ts, starts.data_ptr(), cu_tokens.data_ptr(), rotations.data_ptr(), rs[0], of[0],
                     at, entries, tokens, requests, heads, kv_heads, of[1], 1 if interleaved else 0, 1 if dtype == _TYPES[1] else 0)
    return out


def keep(k_pool, v_pool, table, starts, ids, cu_ids):
    """Moves rows of K and V within requests: position starts[r] + i takes what position
    starts[r] + ids[cu_ids[r] + i] held before the call, for i < cu_ids[r + 1] - cu_ids[r].
    The ids of a request ascend (accepted drafts, numbered from the first one behind
    the context): each is at least its own index, others are not moved.  Requests that
    start below zero, positions past the table and pages outside the pool are skipped;
    pages that rows move in belong to one request.

    table: [requests, entries] int32, starts: [requests], ids: [count], cu_ids:
    [requests + 1] int32."""
    _lib.require_gpu(k_pool, v_pool, table, starts, ids, cu_ids)
    dtype, pages, kv_heads, pools = _pools(k_pool, v_pool)
    requests, entries, ts = _table(table)
    _vector("starts", starts, requests)
    _vector("ids", ids, ids.numel())
    _vector("cu_ids", cu_ids, requests + 1)
    _lib.call_packed("v1_paged_keep", k_pool, *pools, table.data_ptr(), ts, starts.data_ptr(), ids.data_ptr(), cu_ids.data_ptr(),
                     entries, ids.shape[0], requests, kv_heads)


def _attend(q, k_pool, v_pool, table, lens, cu_q, max_q, scale, softcap, slopes, window, prefix, document, parents, out, return_lse):
    _lib.require_gpu(q, k_pool, v_pool, table, lens, cu_q, slopes, prefix, document, parents, out)
    dtype, pages, kv_heads, pools = _pools(k_pool, v_pool)
    qs = _rows("q", q, dtype, None, None)
    tokens, heads, _ = q.shape
    group = heads // kv_heads
    if not heads or heads % kv_heads:
        raise ValueError("query heads must be a multiple of KV heads")
    requests, entries, ts = _table(table)
    if entries * PAGE >= 1 << 31:
        raise ValueError("positions must stay below 2**31")
    _vector("lens", lens, requests)
    cu = 0
    if cu_q is None:
        if tokens != requests:
            raise ValueError("q must hold one query of each request where there is no cu_q")
        max_q = 1
    else:
        _vector("cu_q", cu_q, requests + 1)
        cu = cu_q.data_ptr()
        max_q = tokens if max_q is None else min(int(max_q), tokens)
        if max_q < 0:
            raise ValueError("max_q must not be negative")
    of_prefix = of_document = of_parents = of_slopes = 0
    if prefix is not None:
        _vector("prefix", prefix, requests)
        of_prefix = prefix.data_ptr()
    if document is not None:
        _vector("document", document, tokens)
        of_document = document.data_ptr()
    if parents is not None:
        if max_q > MOST_DRAFTS:
            raise ValueError(f"max_q must be given, at most {MOST_DRAFTS}, for more drafted tokens than that")
        _vector("parents", parents, tokens)
        of_parents = parents.data_ptr()
    if slopes is not None:
        if slopes.dtype != _F32 or slopes.shape != (heads,) or not slopes.is_contiguous():
            raise ValueError(f"slopes must be a contiguous float32 [{heads}] tensor")
        of_slopes = slopes.data_ptr()
    scale = _DEFAULT_SCALE if scale is None else float(scale)
    if not 0.0 < scale < math.inf:
        raise ValueError("softmax_scale must be positive and finite")
    softcap, window = float(softcap), int(window)
    if not 0.0 <= softcap < math.inf:
        raise ValueError("softcap must be finite and not negative")
    if not 0 <= window < 1 << 31:
        raise ValueError("window must be in [0, 2**31)")
    if out is None:
        out = q.new_empty((tokens, heads, DIM))
    os = _rows("out", out, dtype, tokens, heads)
    lse = q.new_empty((tokens, heads), dtype=_F32) if return_lse else None
    # (the sums of a request's parts are the call's own, as in attention.attend_slots)
    ws_bytes = _workspace_bytes(q.get_device(), tokens, requests, kv_heads, group, max_q, entries * PAGE if pages else 0, window)
    ws = q.new_empty((ws_bytes,), dtype=torch.uint8) if ws_bytes else None
    _lib.call_packed("v1_paged_attend", q, q.data_ptr(), qs[0], qs[1], *pools, table.data_ptr(), ts, lens.data_ptr(), cu, of_prefix,
                     of_document, of_parents, of_slopes, out.data_ptr(), os[0], os[1], _lib.ptr(lse), _lib.ptr(ws), ws_bytes,
                     entries, tokens, requests, max_q, kv_heads, group, window, 1 if dtype == _TYPES[1] else 0, scale, softcap)
    return (out, lse) if return_lse else out


def attend(q, k_pool, v_pool, table, lens, cu_q=None, max_q=None, softmax_scale=None, softcap=0.0, slopes=None, window=0, prefix=None,
           document=None, out=None, return_lse=False):
    """Attention of each request's queries over its pages, causal:
    S[i, j] = softmax_scale q_i . k_j, then softcap tanh(S / softcap) where softcap > 0,
    then less slopes[h] |pos - j|; out[i] = sum_j softmax_j(S[i, :]) v_j over the keys seen.
    Query head h reads KV head h // (heads / kv_heads).

    q:      [tokens, heads, 128] of the pools' type
    table:  [requests, entries] int32
    lens:   [requests] int32, each request's keys, its queries' own among them (taken
            within the table's positions): query i of nq has position lens[r] - nq + i
    cu_q:   [requests + 1] int32, where each request's queries begin and end; None: one
            query for each request
    max_q:  at least the longest request's queries; None: tokens.  The first max_q
            queries of a longer one are computed
    softcap: finite, 0: none
    slopes: [heads] fp32
    window: a query sees the last `window` positions up to its own; 0: all
    prefix: [requests] int32, the first positions of a request that all of its queries
            see, whatever the rest says (a prefix that sees itself both ways, or the
            positions a window keeps)
    document: [tokens] int32, the first position that a query sees (where its document
            begins)

    Keys in pages outside the pool are not attended.  A query without keys gives zeros
    and -inf, one whose keys all score -inf NaN and -inf; rows of `out` outside
    [cu_q[0], cu_q[-1]) or past a request's first max_q are left as they are (their
    log-sum-exps are not set).  softmax_scale > 0, default 1 / sqrt(128).  Returns out
    [tokens, heads, 128], and with return_lse the natural log of the sum of
    exponentials, [tokens, heads] fp32."""
    return _attend(q, k_pool, v_pool, table, lens, cu_q, max_q, softmax_scale, softcap, slopes, window, prefix, document, None, out,
                   return_lse)


def attend_tree(q, k_pool, v_pool, table, lens, parents, cu_q=None, max_q=None, softmax_scale=None, softcap=0.0, slopes=None, window=0,
                out=None, return_lse=False):
    """Attention of drafted tokens behind a context: each sees the context, its ancestors
    and itself.  Arguments, scores and results as in `attend`, and

    q:       the drafted tokens' queries; request r's nq of them are the last nq of its
             lens[r] keys, whose first lens[r] - nq are the context
    parents: [tokens] int32: the parent of a draft among its request's, numbered from 0,
             below the draft's own number; others (-1): it follows the context
    max_q:   at least the longest request's drafts, 256 at most; None: tokens

    A draft's position is the context's length plus its depth: `slopes` and `window`
    count from it, a window hides positions of the context alone."""
    if parents is None:
        raise ValueError("parents must be a contiguous int32 tensor")
    return _attend(q, k_pool, v_pool, table, lens, cu_q, max_q, softmax_scale, softcap, slopes, window, None, None, parents, out,
                   return_lse)
