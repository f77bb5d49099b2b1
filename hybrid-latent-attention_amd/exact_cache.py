"""Whole exact caches on MI355X: attention of new tokens over all rows of a paged per-head K / V cache, and the store into it.

The S6 path reads exact K / V in a window of a few rows. Layers and loops that keep their exact cache, and the teacher that a
latent model is measured against, attend to all of it: ``attention`` does, for single tokens and chunks, with any number of query
heads per KV head, and ``store_rows`` writes the rows of new tokens.

A cache is ``[num_blocks, KV heads, block, 2d]`` (K then V, the layout of the exact window; any strides, the last one 1), ``d`` 64,
128 or 256, in bf16 or in ``torch.float8_e4m3fn``. The values of an e4m3 cache count times a scale per KV head (``k_scale``,
``v_scale``: fp32 ``[KV heads]``; None: 1). A page has any number of rows.

Checks, streams and errors are those of ``compact_cache``.
"""
from __future__ import annotations

import torch

from . import _lib, s6_ops
from .compact_cache import _call, _same_device, _table, _vector

BF16, E4M3, F32, I32, I64 = torch.bfloat16, torch.float8_e4m3fn, torch.float32, torch.int32, torch.int64
DIMS = (64, 128, 256)
MAX_SHARES = 1024
# Rows from which tokens alone, in a step with groups of tokens, are cut in shares. A workgroup streams a row in 20 ns, 4096 in 80 us; the
# three launches more take 8 to 12. us with / without, 8 KV heads for 32: one token of 131,000 rows beside 512 tokens on 8160 rows
# 405 / 2670, 16 tokens of 8160 beside 2048 tokens 730 / 950, 8 of 65,000 beside 512 tokens on 4000 440 / 2720; nothing but chunks
# of 512 on 8160 rows 712 / 701.
LONG_ROWS = 4096


def _cache(cache, k_scale, v_scale):
    """``(KV heads, d, e4m3, page, head and row stride, block, pages)`` of an exact cache, checked."""
    shape, stride = cache.shape, cache.stride()
    if cache.dtype != BF16 and cache.dtype != E4M3:
        raise ValueError(f'an exact cache is bfloat16 or float8_e4m3fn, got {cache.dtype}')
    if len(shape) != 4 or shape[3] % 2 or shape[3] // 2 not in DIMS:
        raise ValueError(f'an exact cache is [num_blocks, KV heads, block, 2d] with d in {DIMS}, got {tuple(shape)}')
    if not shape[1]:
        raise ValueError('an exact cache has at least one KV head')
    if stride[3] != 1:
        raise ValueError('an exact cache needs a unit last-dim stride')
    e4m3 = cache.dtype == E4M3
    for name, scale in (('k_scale', k_scale), ('v_scale', v_scale)):
        if scale is not None:
            if not e4m3:
                raise ValueError(f'{name} belongs to a float8_e4m3fn cache, got {cache.dtype}')
            if scale.dtype != F32 or tuple(scale.shape) != (shape[1],) or not scale.is_contiguous():
                raise ValueError(f'{name} must be contiguous fp32 [{shape[1]}], got {scale.dtype} {tuple(scale.shape)}')
    return shape[1], shape[3] // 2, e4m3, stride[0], stride[1], stride[2], shape[2], shape[0]


def store_rows(key, value, slots, cache, k_scale=None, v_scale=None):
    """``key`` and ``value`` (bf16 ``[T, KV heads, d]``, any token and head strides) into slots (int64 ``[T]``, ``page * block +
    row``) of an exact cache; slots outside the cache are skipped, and the slots of a call must differ.

    Into an e4m3 cache goes ``x / scale`` (fp32), clamped to +-448 and rounded to the nearest value, ties to the even one; NaN
    stays NaN."""
    _same_device(cache, key, value, slots, k_scale, v_scale)
    kv_heads, d, e4m3, page, head, row, block, pages = _cache(cache, k_scale, v_scale)
    s6_ops._bf16('key', key)
    s6_ops._bf16('value', value)
    if key.dim() != 3 or key.shape != value.shape or key.shape[1] != kv_heads or key.shape[2] != d:
        raise ValueError(f'key and value must be [T, {kv_heads}, {d}] alike, got {tuple(key.shape)} and {tuple(value.shape)}')
    T = key.shape[0]
    slots = _vector('slots', slots, T, I64)
    _call('hla_s6_exact_store', cache.device, key.data_ptr(), key.stride(0), key.stride(1), value.data_ptr(), value.stride(0),
          value.stride(1), T, kv_heads, d, slots.data_ptr(), _lib.ptr(k_scale), _lib.ptr(v_scale), cache.data_ptr(), int(e4m3),
          page, head, row, block, pages)


def row_shares(max_rows, groups, parts, cu_count=256):
    """``shares`` of ``attention`` for rows of at most ``max_rows`` and ``groups`` (token, KV head) pairs over ``parts`` KV heads: two
    workgroups per CU together, which is what fits one at a time (32 tokens of 1000 to 8160 rows on 8 KV heads: 115 us with a half
    of them, 101, 102 with twice as many), or 0, a workgroup per group, where the second launch costs more than it evens out: on
    short rows, and where the groups are many and no row lasts longer than the others. GPU time in us with shares / a workgroup per
    group, 8 KV heads:

        tokens x rows   1 x 512     1 x 768     1 x 1024    4 x 1024    16 x 1024   16 x 1536   32 x 1536   64 x 1024
                        10.8 / 8.9  10.9 / 10.7 10.9 / 11.2 11.4 / 13.5 19.7 / 17.5 25.1 / 23.6 41.8 / 35.0 51.9 / 47.6

    (a call on the host takes 16 / 11), and with 256 tokens, 16 KV heads:

        rows            256 x 2000  256 x 4000   256 x 8160   1000 to 8160  one of 16000, else 1000  of 32000   of 131000
                        626 / 632   1284 / 1264  2594 / 2573  1459 / 1468   365 / 505                397 / 676  500 / 1735

    (512 tokens of 100 to 2000 rows: 815 / 728). A place takes ``groups / (2 * cu_count)`` of them one behind the other, with 512 rows
    on average as many as the longest may have. A function of constants and the row count only (graph-stable)."""
    if max_rows <= (1536 if 2 * groups >= cu_count else 1024) or (groups >= 16 * cu_count and 256 * groups >= max_rows * cu_count):
        return 0
    return _shares(parts, cu_count)


def _shares(parts, cu_count):
    return max(1, min(MAX_SHARES, 2 * cu_count // parts))


def _turns(tokens, heads, kv_heads, cu_count=256, per_request=1):
    """0, or the workgroups per group of ``16 // heads`` tokens (``heads`` query heads per KV head; the kernel takes ``32 // heads``
    where groups are many) that go through rows together, where there is a group for every CU. Chunks on top of histories, us with
    groups / a workgroup per token: 4 x 512 tokens on 8160 rows of 16 heads 398 / 5861, of 8 KV heads for 32 685 / 2939 (in e4m3 591
    with groups), a prompt of 4000 of 16 heads 235 / 3219, 8 x 64 on 4000 (8 KV heads for 32) 103 / 397.

    A group of single tokens (which a step may have beside its chunks) has as many requests as tokens: with few tokens per request
    on average (``per_request``, at least) a workgroup for each; else 4, since most find nothing to do (a prompt of 4000 with 16: 260)."""
    if heads > 8 or -(-tokens // (16 // heads)) * kv_heads < cu_count:
        return 0
    return 16 // heads if per_request < 32 else min(4, 16 // heads)


def _most_alone(tokens, requests, max_query_len):
    """How many tokens of a step can be the only ones of their request, where the longest has ``max_query_len`` (2 or more)."""
    return max(0, min(tokens - max_query_len, (requests * max_query_len - tokens) // (max_query_len - 1)))


def attention(q, cache, block_table, ctx, scale, max_seq_len, token_requests=None, window=0, k_scale=None, v_scale=None,
              shares=None, workspace=None, max_query_len=None):
    """Attention of ``q [T, H, d]`` (bf16, any token and head strides) over the rows ``[max(0, n - window), n)`` of ``n = ctx[t]``
    (int32; ``window`` 0: over all ``n``) of an exact cache: ``(o [T, H, d] bf16, lse [H, T] fp32)``. ``H`` is a multiple of the
    cache's KV heads, and query head ``h`` reads KV head ``h // (H / KV heads)``. Tokens without rows give ``o = 0``, ``lse = -inf``.

    The rows of a token are those before it and its own, once ``store_rows`` has written it; tokens of one request (a chunk) have a
    ``ctx`` of their own each. ``block_table`` (int32) is per token, or per request with ``token_requests[t]`` (int64) naming the
    row of token ``t``. Tokens of a request that lie one behind the other go through its rows together in large steps of chunks:
    ``max_query_len`` (a host number, the most tokens of a request) defaults to the tokens per row of the table; with a table that has
    rows to spare (a pool's) the tokens would be taken for single ones, 15 times slower in large chunks: pass it. No entry of ``ctx``
    should be above ``max_seq_len`` (a host number, which sets how rows are cut). Scores, softmax statistics and sums are fp32; weights
    keep 16 bits in their product with V.

    The rows of all tokens are cut in ``shares`` equal parts per KV head (0: a workgroup takes all rows of a token; defaults to
    ``row_shares``); their partial results go through ``workspace`` (an ``S6Workspace`` of ``2 * shares * H * (d + 1) + 2 * T`` floats;
    defaults to a new buffer). Calls that share a workspace must not overlap. Beside chunks, tokens that are the only ones of their
    request are cut in shares where rows are long (``LONG_ROWS``); a workspace without room for that, ``T + 1`` floats more, is not used."""
    _same_device(cache, q, block_table, ctx, token_requests, k_scale, v_scale)
    kv_heads, d, e4m3, page, head, row, block, pages = _cache(cache, k_scale, v_scale)
    s6_ops._bf16('q', q)
    shape = q.shape
    if len(shape) != 3 or shape[2] != d or shape[1] % kv_heads or not shape[1]:
        raise ValueError(f'q must be [T, a multiple of {kv_heads} heads, {d}], got {tuple(shape)}')
    T, H, _ = shape
    ctx = _vector('ctx', ctx, T)
    table_stride, cols, count = _table(block_table, T if token_requests is None else min(T, 1))
    if token_requests is not None:
        token_requests = _vector('token_requests', token_requests, T, I64)
    window = int(window)
    if window < 0:
        raise ValueError(f'window must not be negative, got {window}')
    dev = q.device
    longest = min(int(max_seq_len), cols * block, window or cols * block)
    parts = kv_heads * -(-H // kv_heads // 16)
    cus = _lib.device_cus(dev.index)
    turns, chunk = 0, 1
    if token_requests is not None:
        chunk = T // max(1, count) if max_query_len is None else int(max_query_len)
    if shares is None:
        if chunk >= 4:
            turns = _turns(T, H // kv_heads, kv_heads, cus, T // max(1, min(count, T - chunk + 1)))   # (most requests there can be)
        if not turns:
            shares = row_shares(longest, T * parts, parts, cus)
        else:   # those of tokens alone
            alone = count - 1 if max_query_len is None else _most_alone(T, count, chunk)
            shares = _shares(parts, cus) if longest >= LONG_ROWS and alone else 0
    else:
        shares = int(shares)
    if not 0 <= shares <= MAX_SHARES:
        raise ValueError(f'shares must be 0 to {MAX_SHARES}, got {shares}')
    ws = None
    if shares:
        need = 2 * shares * H * (d + 1) + (3 * T + 1 if turns else 2 * T)
        ws = None if workspace is None else workspace.ensure(dev)
        if ws is None or (turns and ws.numel() < need):
            ws = torch.empty(need, dtype=F32, device=dev)
        if ws.numel() < need:
            raise RuntimeError(f'S6 workspace overflow: need {need} floats, have {ws.numel()}')
        _same_device(q, ws)   # (a workspace keeps the device of its first use)
    out = torch.empty(T, H, d, dtype=BF16, device=dev)
    lse = torch.empty(H, T, dtype=F32, device=dev)
    token_stride, head_stride, _ = q.stride()
    _call('hla_s6_exact_attention', dev, q.data_ptr(), T, H, d, token_stride, head_stride, cache.data_ptr(), int(e4m3), kv_heads,
          page, head, row, block, pages, block_table.data_ptr(), table_stride, cols, count, _lib.ptr(token_requests),
          ctx.data_ptr(), window, float(scale), _lib.ptr(k_scale), _lib.ptr(v_scale), shares, turns, _lib.ptr(ws),
          0 if ws is None else ws.numel(), out.data_ptr(), H * d, d, lse.data_ptr(), int(chunk > 1))
    return out, lse
