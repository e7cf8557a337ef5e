"""Latent K/V cache and its attention: the consumer of the indexer's Top-K slots
where one latent vector per token serves every head.

A cache row is 656 bytes: 512 OCP e4m3fn codes, 64 bf16 rope-key numbers, 4 fp32
scales, in this order (code j stands for code * scale[j // 128]; a cache with its
scales before the rope numbers is another format of the same size, and is not told
apart); the row that native_kernels.gather_rows, the page manager and the tail
staging move as opaque bytes.  `store_rows` writes rows, `attend` reads them with
queries that already carry the key projection ("absorbed": one key of 512 + 64
numbers for all heads, its first 512 the value), `attend_expanded` is the prompt's
form over keys and values expanded per head from the latent.

Sums are fp32, undivided until the end, and may carry 2^16 times the keys' number
times a value: they are kept for magnitudes between 2^-100 and 2^100.

Every call launches on the current stream of its tensors' device, never
synchronises, and raises ValueError for arguments that do not fit.
"""
import functools
import math

import torch

from . import _lib

LATENT, ROPE, ROW_BYTES = 512, 64, 656
HEAD = 128  # key numbers of a head beside the rope's, and value numbers, in the expanded form


_BF16, _I32 = torch.bfloat16, torch.int32


def _int32(name, t, n):
    if t.dtype != _I32 or t.shape != (n,) or not t.is_contiguous():
        raise ValueError(f"{name} must be a contiguous int32 tensor of shape [{n}]")


# (each property of a tensor is asked for once: 0.1-0.3 us of a call whose kernels
# may take 10)
def _pool(pool):
    """Rows and their stride."""
    shape, stride = pool.shape, pool.stride()
    if pool.dtype != torch.uint8 or len(shape) != 2 or shape[1] != ROW_BYTES or stride[1] != 1:
        raise ValueError(f"pool must be a uint8 [rows, {ROW_BYTES}] tensor with unit inner stride")
    return shape[0], stride[0]


def _output(out, q, shape):
    """The output and its strides."""
    if out is None:
        out = q.new_empty(shape)
    stride = out.stride()
    if out.dtype != _BF16 or out.shape != shape or stride[2] != 1:
        raise ValueError(f"out must be bfloat16 {list(shape)} with a contiguous last dimension")
    return out, stride[0], stride[1]


_DEFAULT_SCALE = 1.0 / math.sqrt(HEAD + ROPE)


def _scale(softmax_scale):
    scale = _DEFAULT_SCALE if softmax_scale is None else float(softmax_scale)
    if not 0.0 < scale < math.inf:
        raise ValueError("softmax_scale must be positive and finite")
    return scale


# (sizes alone decide: asked of the library once for each)
@functools.lru_cache(maxsize=4096)
def _workspace_bytes(entry, index, *sizes):
    return _lib.workspace_bytes(entry, index, *sizes)


def store_rows(latent, rope, pool, slots):
    """Writes token t's row into pool[slots[t]] (a slot below zero or past the
    pool: the token is skipped; slots of one call are distinct, or which token's
    bytes a row holds is undefined).

    latent: [tokens, 512] bf16, rope: [tokens, 64] bf16, pool: [rows, 656] uint8
    (row strides free), slots: [tokens] int32.  A block's scale is the smallest
    power of two s (2^-126 at least) with |x| <= 448 s for its finite numbers, a
    code the nearest e4m3 value of x / s (ties to even); infinities are stored as
    +-448 s, NaN as NaN."""
    _lib.require_gpu(latent, rope, pool, slots)
    shape, ls, rs = latent.shape, latent.stride(), rope.stride()
    tokens = shape[0] if len(shape) == 2 else -1
    if shape != (tokens, LATENT) or latent.dtype != _BF16 or ls[1] != 1:
        raise ValueError(f"latent must be bfloat16 [tokens, {LATENT}] with a contiguous last dimension")
    if rope.shape != (tokens, ROPE) or rope.dtype != _BF16 or rs[1] != 1:
        raise ValueError(f"rope must be bfloat16 [tokens, {ROPE}] with a contiguous last dimension")
    rows, stride = _pool(pool)
    _int32("slots", slots, tokens)
    _lib.call_packed("v1_latent_store", pool, latent.data_ptr(), ls[0], rope.data_ptr(), rs[0], slots.data_ptr(),
                     pool.data_ptr(), rows, stride, tokens)
    return pool


def attend(q, pool, ids=None, table=None, page_bits=0, lens=None, softmax_scale=None, out=None, return_lse=False):
    """out[r, h] = sum_j softmax_j(scale * (q[r, h, :512] . c_j + q[r, h, 512:] . rope_j)) c_j
    over the keys of row r, c_j the dequantised latent vector.

    q:     [rows, heads, 576] bf16
    pool:  [slots, 656] uint8 (row stride free)
    ids:   [rows, keys] int32 positions (the Top-K's output), or None: positions 0, 1, ...
    table: None (positions are pool rows), a 1-D page table shared by all rows, or
           [rows, entries]; row = (table[r, id >> page_bits] << page_bits) | (id & (2**page_bits - 1)),
           as in native_kernels.gather_rows
    lens:  [rows] int32: the first lens[r] entries of ids (or positions) are row r's; None: all.
           Without ids and lens every position of the table (or pool) is attended.

    Ids below zero, past the table or outside the pool are not attended.  A row
    without keys gives zeros and a log-sum-exp of -inf, one whose keys all score
    -inf NaN and -inf.  softmax_scale > 0: default
    1 / sqrt(192), that of the expanded form.  Returns out [rows, heads, 512] bf16,
    and with return_lse the natural log of the sum of exponentials, [rows, heads] fp32."""
    _lib.require_gpu(q, pool, ids, table, lens, out)
    shape, qs = q.shape, q.stride()
    if len(shape) != 3 or shape[2] != LATENT + ROPE or q.dtype != _BF16 or qs[2] != 1 or not shape[1]:
        raise ValueError(f"q must be bfloat16 [rows, heads, {LATENT + ROPE}] with a contiguous last dimension")
    slots, slot_stride = _pool(pool)
    rows, heads, _ = shape
    page_bits = int(page_bits)
    if not 0 <= page_bits < 31:
        raise ValueError("page_bits must be in [0, 31)")
    map_ptr = map_len = map_stride = ids_ptr = ids_stride = lens_ptr = 0
    if table is not None:
        of, at = table.shape, table.stride()
        dims = len(of)
        if table.dtype != _I32 or not (dims == 1 or (dims == 2 and of[0] == rows)):
            raise ValueError("table must be int32 [entries] or [rows, entries]")
        map_ptr, map_len, map_stride = table.data_ptr(), of[-1], at[0] if dims == 2 else 0
        if map_len and at[-1] != 1:
            raise ValueError("table must have unit inner stride")
    if ids is not None:
        of, at = ids.shape, ids.stride()
        if ids.dtype != _I32 or len(of) != 2 or of[0] != rows or (at[1] != 1 and of[1]):
            raise ValueError("ids must be int32 [rows, keys] with unit inner stride")
        keys, ids_ptr, ids_stride = of[1], ids.data_ptr(), at[0]
    else:
        keys = map_len << page_bits if table is not None else slots
        if keys >= 1 << 31:
            raise ValueError("positions must stay below 2**31")
    if table is not None and map_len == 0:
        keys = 0
    if lens is not None:
        _int32("lens", lens, rows)
        lens_ptr = lens.data_ptr()
    scale = _scale(softmax_scale)
    out, o_row, o_head = _output(out, q, (rows, heads, LATENT))
    lse = q.new_empty((rows, heads), dtype=torch.float32) if return_lse else None
    # (the sums of a row's parts are the call's own, as in attention.attend_slots)
    ws_bytes = _workspace_bytes("v1_latent_attend_workspace", q.get_device(), rows, heads, keys, lens is not None)
    ws = q.new_empty((ws_bytes,), dtype=torch.uint8) if ws_bytes else None
    _lib.call_packed("v1_latent_attend", q, q.data_ptr(), qs[0], qs[1], pool.data_ptr(), slots, slot_stride, map_ptr, map_len,
                     map_stride, ids_ptr, ids_stride, lens_ptr, out.data_ptr(), o_row, o_head, _lib.ptr(lse), _lib.ptr(ws),
                     ws_bytes, page_bits, rows, heads, keys, scale)
    return (out, lse) if return_lse else out


def attend_expanded(q, kv, k_rope, cu_q, cu_k=None, max_q=None, softmax_scale=None, causal=True, out=None,
                    return_lse=False):
    """Attention of a batch of sequences laid end to end, over keys and values
    expanded per head from the latent:
    S[i, j] = scale * (q[i, h, :128] . kv[j, h, :128] + q[i, h, 128:] . k_rope[j]),
    out[i, h] = sum_j softmax_j(S[i, j]) kv[j, h, 128:].

    q:      [tokens, heads, 192] bf16
    kv:     [keys, heads, 256] bf16 (128 key numbers, then 128 value numbers: the
            up-projection's output as it is)
    k_rope: [keys, 64] bf16, every head's
    cu_q, cu_k: [batch + 1] int32, where each sequence's queries and keys begin and
            end (cu_k None: cu_q).  With `causal`, query i of nq sees keys
            j <= nk - nq + i of its nk (a chunk at the end of its context), else all.
    max_q:  at least the longest sequence's queries; None: tokens.  The first max_q
            queries of a longer one are computed, their keys counted from its end as ever.

    A query without keys gives zeros and -inf, one whose keys all score -inf NaN
    and -inf; rows of `out` outside [cu_q[0], cu_q[-1]) or past a sequence's first
    max_q are left as they are (their log-sum-exps are not set).  softmax_scale > 0, default 1 / sqrt(192).  Returns
    out [tokens, heads, 128] bf16, and with return_lse the natural log of the sum
    of exponentials, [tokens, heads] fp32."""
    cu_k = cu_q if cu_k is None else cu_k
    _lib.require_gpu(q, kv, k_rope, cu_q, cu_k, out)
    if q.dim() != 3 or q.shape[2] != HEAD + ROPE or q.dtype != _BF16 or q.stride(2) != 1 or not q.shape[1]:
        raise ValueError(f"q must be bfloat16 [tokens, heads, {HEAD + ROPE}] with a contiguous last dimension")
    tokens, heads, _ = q.shape
    keys = kv.shape[0] if kv.dim() == 3 else -1
    if kv.dtype != _BF16 or kv.shape != (keys, heads, 2 * HEAD) or kv.stride(2) != 1:
        raise ValueError(f"kv must be bfloat16 [keys, heads, {2 * HEAD}] with a contiguous last dimension")
    if k_rope.dtype != _BF16 or k_rope.shape != (keys, ROPE) or k_rope.stride(1) != 1:
        raise ValueError(f"k_rope must be bfloat16 [keys, {ROPE}] with a contiguous last dimension")
    batch = cu_q.numel() - 1
    if cu_q.dim() != 1 or batch < 0:
        raise ValueError("cu_q must be a contiguous int32 [batch + 1] tensor")
    _int32("cu_q", cu_q, batch + 1)
    _int32("cu_k", cu_k, batch + 1)
    max_q = tokens if max_q is None else min(int(max_q), tokens)
    if max_q < 0:
        raise ValueError("max_q must not be negative")
    scale = _scale(softmax_scale)
    out, o_row, o_head = _output(out, q, (tokens, heads, HEAD))
    lse = q.new_empty((tokens, heads), dtype=torch.float32) if return_lse else None
    ws_bytes = _workspace_bytes("v1_latent_expanded_workspace", q.get_device(), tokens, keys, batch, heads, max_q)
    ws = q.new_empty((ws_bytes,), dtype=torch.uint8) if ws_bytes else None
    q_row, q_head, _ = q.stride()
    _lib.call_packed("v1_latent_expanded", q, q.data_ptr(), q_row, q_head, kv.data_ptr(), kv.stride(0),
                     kv.stride(1), k_rope.data_ptr(), k_rope.stride(0), cu_q.data_ptr(), cu_k.data_ptr(), out.data_ptr(),
                     o_row, o_head, _lib.ptr(lse), _lib.ptr(ws), ws_bytes, tokens, keys, batch, heads, max_q,
                     1 if causal else 0, scale)
    return (out, lse) if return_lse else out
