"""The compact latent cache on MI355X: latent rows in 4 bits per value, attention over them, and eviction.

A compact cache takes the place of a ``[num_blocks, 1, block, 2w]`` bf16 latent cache where HBM capacity or bandwidth is
what a step waits for: it is a uint8 tensor ``[num_blocks, block / 16, 17 w]`` (``cache_shape``), 4.25 bits per value. Values
are E2M1 numbers (0, 0.5, 1, 1.5, 2, 3, 4, 6 and their negatives) times a power of two shared by 32 columns; the bytes of a
tile of 16 rows lie in the order in which the matrix instructions read them (``csrc/compact.h``). Block tables, slots and
lengths are those of the bf16 cache.

``store_rows`` and ``load_rows`` move rows in and out, ``history_attention`` (or ``history_partials`` with
``s6_ops.split_epilogue``) attends to them; ``s6_layer.attend``, ``write_commit`` and ``store_rows`` take a compact cache where
they take a bf16 one.

Eviction works on both kinds of cache: ``attention_weights`` adds what a step's attention gave every row to an account,
``select_rows`` picks the rows that stay, ``move_rows`` brings them together at the front of each request's pages.

Checks, streams and errors are those of ``s6_ops``: tensors on the GPU (``RuntimeError`` otherwise), shapes and types
refused with ``ValueError`` before any launch, everything enqueued on the current stream of the tensors' device, nothing
synchronised, every call capturable in a HIP graph.
"""
from __future__ import annotations

from collections import namedtuple

import torch

from . import _lib, s6_ops

BF16, F32, I32, I64, U8 = torch.bfloat16, torch.float32, torch.int32, torch.int64, torch.uint8
WIDTHS = (128, 256, 512, 1024)
HEADS, TILE = 16, 16
# rows from which a history is long enough to be cut between workgroups in steps that could do without
LONG_ROWS = 4096
# rows of all requests up to which a step may expand them to bf16: 256 MiB of scratch at width 512
EXPANDED_ROWS = 1 << 17

#: What ``select_rows`` returns. ``lengths [R]``: rows per request from now on; ``weights``, ``positions [R, M]``: the account
#: and positions in the new order (0 and -1 behind the last row); ``source``, ``target [R, M // 2]``: the row moves, ended by -1.
Eviction = namedtuple('Eviction', 'lengths weights positions source target')


def _call(name, device, *args):
    """One entry point on the current stream of ``device``, whichever device is current."""
    if device.index == torch.cuda.current_device():
        _lib.call(name, *args, _lib.stream(device))
    else:
        with torch.cuda.device(device):
            _lib.call(name, *args, _lib.stream(device))


def _same_device(first, *others):
    at = first.get_device()   # below 0 on the host
    for t in others:
        if t is not None and t.get_device() != at:
            break
    else:
        if at >= 0:
            return
    s6_ops._dev(first, *others)
    for t in others:
        if t is not None and t.device != first.device:
            raise RuntimeError(f'tensors on {first.device} and {t.device}')


def _width(w):
    if w not in WIDTHS:
        raise ValueError(f'latent width {w} not in {WIDTHS}')
    return w


def cache_shape(num_blocks, block_size, width):
    """Shape of a compact cache (uint8) of ``num_blocks`` pages of ``block_size`` rows of ``2 * width`` values."""
    if block_size <= 0 or block_size % TILE:
        raise ValueError(f'block size {block_size} is not a positive multiple of {TILE}')
    return int(num_blocks), block_size // TILE, 17 * _width(width)


def is_compact(cache):
    """Whether ``cache`` is a compact cache (uint8) rather than a bf16 one."""
    return cache is not None and cache.dtype == U8


def block_size(cache):
    """Rows per page of a compact cache."""
    return cache.shape[1] * TILE


def _compact(cache, width=None):
    """``(width, page stride, block, pages)`` of a compact cache, checked."""
    if cache.dtype != U8:
        raise ValueError(f'a compact cache is uint8, got {cache.dtype}')
    shape, stride = cache.shape, cache.stride()
    if len(shape) != 3 or shape[2] % 17 or (width is not None and shape[2] != 17 * width):
        raise ValueError(f'compact cache must be [num_blocks, block / 16, {17 * width if width else "17 w"}], '
                         f'got {tuple(shape)}')
    if stride[2] != 1 or (shape[1] > 1 and stride[1] != shape[2]):
        raise ValueError('the pages of a compact cache must be contiguous')
    return _width(shape[2] // 17), stride[0], shape[1] * TILE, shape[0]


def _table(block_table, rows):
    """``(row stride, columns, rows)`` of a block table of at least ``rows`` rows, checked."""
    stride = block_table.stride()
    if block_table.dtype != I32 or len(stride) != 2 or stride[1] != 1:
        raise ValueError('block_table must be a 2-d int32 tensor with a unit last stride')
    count, cols = block_table.shape
    if count < rows:
        raise ValueError(f'block_table has {count} rows, {rows} are needed')
    return stride[0], cols, count


def _vector(name, t, n, dtype=I32):
    if t.shape != (n,):
        raise ValueError(f'{name} must have {n} entries, got {tuple(t.shape)}')
    if t.dtype != dtype:
        raise ValueError(f'{name} must be {dtype}, got {t.dtype}')
    return t if t.is_contiguous() else t.contiguous()


def _rows2d(name, t, dtype, shape=None):
    """``(row stride, columns)`` of a 2-d tensor, checked."""
    stride = t.stride()
    if t.dtype != dtype or len(stride) != 2 or stride[1] != 1 or (shape is not None and t.shape != shape):
        want = '' if shape is None else f' {list(shape)}'
        raise ValueError(f'{name} must be a 2-d {dtype} tensor{want} with a unit last stride, got {t.dtype} {list(t.shape)}')
    return stride[0], t.shape[1]


def _query(q, width=None):
    s6_ops._bf16('q_lat', q)
    shape = q.shape
    if len(shape) != 3 or shape[1] != HEADS:
        raise ValueError(f'q_lat must be [T, {HEADS}, width], got {tuple(shape)}')
    if width is not None and shape[2] != width:
        raise ValueError(f'q_lat has width {shape[2]}, the cache {width}')
    return shape[0], shape[2]


# ----------------------------------------------------------------------------------------------------------------
# Rows in and out
# ----------------------------------------------------------------------------------------------------------------

def store_rows(key, value, slots, cache):
    """Quantise ``[key | value]`` rows (``[T, w]`` bf16 each, any row stride) into slots (int64 ``[T]``, ``page * block +
    row``) of a compact cache; slots outside the cache are skipped, and the slots of a call must differ.

    Per 32 columns the scale is the smallest power of two ``s`` with ``max|x| <= 7 s`` (so the largest value goes to its nearest
    neighbour), exponent -120 to 125; values go to the nearest E2M1 number, ties to the even one. 32 columns with an
    infinity or NaN among them read as NaN."""
    _same_device(cache, key, value, slots)
    s6_ops._bf16('key', key)
    s6_ops._bf16('value', value)
    if key.dim() != 2 or key.shape != value.shape:
        raise ValueError(f'key and value must be [T, w] alike, got {tuple(key.shape)} and {tuple(value.shape)}')
    T, w = key.shape
    _, page_stride, block, pages = _compact(cache, w)
    slots = _vector('slots', slots, T, I64)
    _call('hla_s6_compact_store', cache.device, key.data_ptr(), key.stride(0), value.data_ptr(), value.stride(0), T, w,
          slots.data_ptr(), cache.data_ptr(), page_stride, block, pages)


def load_rows(cache, block_table, lengths, max_rows, out=None):
    """The rows of requests as bf16: ``[R, max_rows, 2w]`` with rows ``lengths[r]`` (int32 ``[R]``) and on of request ``r``
    zero. ``block_table`` is per request. ``out`` (any request and row strides) is written if given."""
    _same_device(cache, block_table, lengths, out)
    geometry = _compact(cache)
    w, R = geometry[0], lengths.shape[0]
    lengths = _vector('lengths', lengths, R)
    max_rows = int(max_rows)
    if out is None:
        out = torch.empty(R, max_rows, 2 * w, dtype=BF16, device=cache.device)
    else:
        s6_ops._bf16('out', out)
        if tuple(out.shape) != (R, max_rows, 2 * w):
            raise ValueError(f'out must be [{R}, {max_rows}, {2 * w}], got {tuple(out.shape)}')
    _load(cache, geometry, block_table, lengths, None, None, 0, R, max_rows, out)
    return out


def _load(cache, geometry, block_table, lengths, query_start_loc, ctx, T, R, max_rows, out):
    w, page_stride, block, pages = geometry
    table_stride, cols, _ = _table(block_table, R)
    request_stride, row_stride, _ = out.stride()
    _call('hla_s6_compact_load', cache.device, cache.data_ptr(), w, page_stride, block, pages, block_table.data_ptr(),
          table_stride, cols, _lib.ptr(lengths), _lib.ptr(query_start_loc), _lib.ptr(ctx), T, R, max_rows, out.data_ptr(),
          request_stride, row_stride)


# ----------------------------------------------------------------------------------------------------------------
# History attention
# ----------------------------------------------------------------------------------------------------------------

def kv_splits(max_seq_len, num_tokens, cu_count=256, width=512, small_step_tiles=768):
    """Split slots per row for ``history_attention`` over a compact cache, one token a workgroup. A split is a workgroup of
    four waves that walk 128 rows at a time. The plan cuts rows so that about half of the slots get equal work, and this returns
    the count that gives every CU one of them (64 rows of 8160 at width 512: 57.6 us with 8 slots, 62.9 with 16); half of that
    up to 256 rows per CU (128 above width 512), where partials cost more than workgroups gain (8 of 8160: 21.8 us with 32
    slots, 22.8 with 64; 1 of 32736: 18.6 with 256, 21.7 with 512); at most two per 128 keys of the longest row, and in small
    steps two per 64 and one per two CUs (1 of 8160: 14.5 with 128, 15.3 with 256). One slot, without a reduction, for rows that
    a single pass covers and for steps with a row for every other CU (130 rows of 4000: 67.5 us with one slot, 75.5 with two, 81.3
    with four, 67.3 with six; 200 of 200 to 4000: 62.3 with one, 68.3 with four; 128 of 2000: 38.8 with either). On long rows
    four slots pay as long as their items, two per row, are no more than the CUs: 128 of 8160 129 us with one slot, 102 with
    four; 129 of 8160 131 and 144 (six: 119, the most that one slot gives away there; 160 rows 140, 152, 133; 200 161, 171, 176;
    250 175, 196, 207). A function of constants and the row count only (graph-stable)."""
    tokens = max(1, num_tokens)
    if max_seq_len <= 128 or 2 * tokens >= cu_count + (max_seq_len >= LONG_ROWS):
        return 1
    few = tokens * max_seq_len <= cu_count * (256 if width <= 512 else 128)
    slots = (1 if few else 2) * max(1, cu_count // tokens)
    if tokens * -(-max_seq_len // TILE) < small_step_tiles:
        return max(2, min(slots, 2 * -(-max_seq_len // 64), cu_count // 2))
    return max(2, min(slots, 2 * -(-max_seq_len // 128), 1024))


def history_shape(max_seq_len, num_tokens, num_reqs, cu_count=256, width=512):
    """How ``history_attention`` runs a step: ``(kind, split slots)`` with ``kind`` 1 for a token per workgroup, 2 for two
    tokens that share the conversion of their rows (uniform splits, no plan), 3 for rows expanded to bf16 once per request and
    the multi-query kernels of the bf16 cache over them. In us at 1 / 2 / 3, best split counts:

        tokens x rows          w 256             w 512             w 1024
        4 x 512 on 8160        458 / 322 / 403   765 / 668 / 567   2645 / 2025
        4 x 512 on 1000        76 / 54 / 74      115 / 110 / 105   401 / 307
        16 x 128 on 4000       234 / 169 / 215   397 / 353 / 337   1340 / 1025
        1 x 512 on 8160        127 / 95          212 / 194         690 / 512
        1 x 512 on 300         13 / 12           18 / 20           48 / 39
        64 x 8 on 4000         86 / 53           146 / 127         390 / 275
        1 x 256 on 2000        23 / 27           38 / 50           102 / 100
        2 x 64 on 8160         44 / 36           68 / 67           197 / 162
        4 x 8 on 8160          21 / 20           32 / 32           65 / 60
        4 x 3 on 8160          16 / 23           24 / 33           42 / 57
        2 x 64 on 2000         22 / 22           35 / 36           73 / 64

    At width 128 there is a token per workgroup alone (4 x 512 on 8160: 278). So two tokens from 2 per CU
    on, and on long rows from one per 8 CUs on; expansion at width 512 alone, from 8 tokens per CU in chunks of 256 and more on
    average, for up to ``EXPANDED_ROWS`` rows: its scratch stays below 256 MiB where memory is what a compact cache is for.
    (Measured on steps of equal chunks; of others the rule sees averages.)"""
    per_request = num_tokens / max(1, num_reqs)
    if width == 512 and num_tokens >= 8 * cu_count and per_request >= 256 and 0 < num_reqs * max_seq_len <= EXPANDED_ROWS:
        return 3, 1
    if width >= 256 and per_request >= 4:
        if num_tokens >= 2 * cu_count:
            return 2, 1
        if max_seq_len >= LONG_ROWS and 8 * num_tokens >= cu_count:
            return 2, max(4, 2 * cu_count // num_tokens)
    return 1, kv_splits(max_seq_len, num_tokens, cu_count, width)


def _history(q, cache, geometry, block_table, table, ctx, scale, token_requests, splits, workspace, plan, tokens_per_group,
             shared_rows, out):
    """The split kernel, and with ``out`` the reduction; returns ``(lse or None, workspace or None)``."""
    T, _, w = q.shape
    _, page_stride, block, pages = geometry
    token_stride, head_stride, _ = q.stride()
    table_stride, cols, count = table
    dev = q.device
    ws = lse = None
    if splits > 1 or out is None:
        need = T * HEADS * splits * (w + 1)
        ws = (torch.empty(need, dtype=F32, device=dev) if workspace is None
              else workspace.attn_logits(T, HEADS, splits, w, dev))
        _same_device(q, ws)   # (a workspace keeps the device of its first use)
    if out is not None:
        lse = torch.empty(HEADS, T, dtype=F32, device=dev)
    _call('hla_s6_compact_history', dev, q.data_ptr(), T, HEADS, w, token_stride, head_stride, cache.data_ptr(), page_stride,
          block, pages, block_table.data_ptr(), table_stride, cols, count, _lib.ptr(token_requests), ctx.data_ptr(),
          float(scale), splits, _lib.ptr(ws), 0 if ws is None else ws.numel(), _lib.ptr(plan),
          0 if plan is None else plan.numel(), tokens_per_group, int(shared_rows), _lib.ptr(out), HEADS * w, w, _lib.ptr(lse))
    return lse, ws


def _operands(q, cache, block_table, ctx, token_requests, plan=None):
    _same_device(cache, q, block_table, ctx, token_requests, plan)
    T, w = _query(q)
    geometry = _compact(cache, w)
    ctx = _vector('ctx', ctx, T)
    table = _table(block_table, T if token_requests is None else min(T, 1))
    if token_requests is not None:
        token_requests = _vector('token_requests', token_requests, T, I64)
    if plan is not None and (plan.dtype != I32 or plan.dim() != 1 or not plan.is_contiguous()):
        raise ValueError(f'plan must be a contiguous 1-d int32 tensor (s6_ops.split_plan), got {plan.dtype} {list(plan.shape)}')
    return T, w, geometry, table, ctx, token_requests


def history_attention(q_lat, cache, block_table, ctx, scale, max_seq_len, token_requests=None, query_start_loc=None,
                      max_query_len=1, num_kv_splits=None, workspace=None, plan=None):
    """Fully visible attention of ``q_lat [T, 16, w]`` (bf16) over the first ``ctx[t]`` (int32) rows of a compact cache:
    ``(o [T, 16, w] bf16, lse [16, T] fp32)``; tokens without rows give ``o = 0``, ``lse = -inf``.

    ``block_table`` (int32) is per token, or per request with ``token_requests[t]`` (int64) naming the row of token ``t``. No
    entry of ``ctx`` may be above ``max_seq_len`` (a host number: it sets the split count). Scores, softmax statistics and
    sums are fp32; the weights are rounded to bf16 for their product with the rows, as over a bf16 cache.

    Requests of several tokens (``max_query_len`` above 1, a host number) share their rows: with ``token_requests`` two tokens
    may go through a row together, and with ``query_start_loc`` (int32 ``[R + 1]``, of the same requests: a token outside all
    of its chunks may name any) too the rows of large chunks may be expanded to bf16 once, into scratch of ``R * max_seq_len``
    rows (``history_shape`` says when, and up to how many).

    ``num_kv_splits`` defaults to the count of ``history_shape``; ``workspace`` (an ``S6Workspace``) to a new buffer; ``plan`` is
    an optional ``s6_ops.split_plan`` for ``(ctx, columns * block, num_kv_splits)``, for a token per workgroup. Calls that share
    a workspace must not overlap."""
    T, w, geometry, table, ctx, token_requests = _operands(q_lat, cache, block_table, ctx, token_requests, plan)
    max_seq_len = int(max_seq_len)
    kind, splits = _shape(q_lat, table, max_seq_len, token_requests, query_start_loc, max_query_len, plan)
    if num_kv_splits is not None:
        splits = int(num_kv_splits)
    longest = min(max_seq_len, table[1] * geometry[2])
    # (its kernel folds a positive scale)
    if kind == 3 and splits == 1 and query_start_loc is not None and longest > 0 and scale > 0:
        with torch.cuda.device(q_lat.device):
            return _expanded_attention(q_lat, cache, geometry, block_table, ctx, scale, longest, token_requests,
                                       query_start_loc)
    out = torch.empty(T, HEADS, w, dtype=BF16, device=q_lat.device)
    lse, _ = _history(q_lat, cache, geometry, block_table, table, ctx, scale, token_requests, splits, workspace, plan,
                      min(kind, 2), max_query_len > 1, out)
    return out, lse


def _shape(q, table, max_seq_len, token_requests, query_start_loc, max_query_len, plan):
    T, _, w = q.shape
    cus = _lib.device_cus(q.get_device())
    if max_query_len == 1 or token_requests is None or plan is not None:
        return 1, kv_splits(max_seq_len, T, cus, w)
    R = table[2] if query_start_loc is None else query_start_loc.shape[0] - 1
    return history_shape(max_seq_len, T, R, cus, w)


def _expanded_attention(q, cache, geometry, block_table, ctx, scale, longest, token_requests, query_start_loc):
    T, w = q.shape[0], q.shape[2]
    _same_device(cache, query_start_loc)
    R = query_start_loc.shape[0] - 1
    qsl = _vector('query_start_loc', query_start_loc, R + 1)
    pages = -(-longest // TILE)
    rows = torch.empty(R * pages, 1, TILE, 2 * w, dtype=BF16, device=q.device)
    _load(cache, geometry, block_table, None, qsl, ctx, T, R, pages * TILE, rows.view(R, pages * TILE, 2 * w))
    table = torch.arange(R * pages, dtype=I32, device=q.device).view(R, pages)
    return s6_ops.history_attention_kv(q, rows[..., :w], rows[..., w:], table, ctx, scale, 1, None, None, None, s6_ops.HIP,
                                       bt_rows=token_requests.clamp(0, R - 1), tokens_per_group=4, shared_rows=True,
                                       nan_rows=True)


def history_partials(q_lat, cache, block_table, ctx, scale, num_kv_splits, workspace, token_requests=None, plan=None,
                     query_start_loc=None, max_query_len=1, max_seq_len=None):
    """The split kernel of ``history_attention`` alone: its partials in ``workspace``, in the layout that
    ``s6_ops.history_reduce`` and ``s6_ops.split_epilogue`` read (``[T, 16, splits, w + 1]``, private). ``max_seq_len``
    defaults to the rows that a row of the table holds."""
    T, w, geometry, table, ctx, token_requests = _operands(q_lat, cache, block_table, ctx, token_requests, plan)
    if workspace is None:
        raise RuntimeError('history partials need an S6Workspace')
    longest = table[1] * geometry[2] if max_seq_len is None else int(max_seq_len)
    kind, _ = _shape(q_lat, table, longest, token_requests, query_start_loc, max_query_len, plan)
    _, ws = _history(q_lat, cache, geometry, block_table, table, ctx, scale, token_requests, int(num_kv_splits), workspace,
                     plan, min(kind, 2), max_query_len > 1, None)
    return ws


# ----------------------------------------------------------------------------------------------------------------
# Eviction
# ----------------------------------------------------------------------------------------------------------------

def _pages(cache, width=None):
    """Geometry of either kind of cache: ``(width, compact, page_stride, row_stride, block, num_blocks)``."""
    if is_compact(cache):
        w, page_stride, block, pages = _compact(cache, width)
        return w, 1, page_stride, 0, block, pages
    s6_ops._bf16('cache', cache)
    if cache.dim() != 4 or cache.shape[1] != 1 or cache.shape[3] % 2 or (width is not None and cache.shape[3] != 2 * width):
        raise ValueError(f'latent cache must be [num_blocks, 1, block, {2 * width if width else "2 w"}], got {tuple(cache.shape)}')
    return _width(cache.shape[3] // 2), 0, cache.stride(0), cache.stride(2), cache.shape[2], cache.shape[0]


def attention_weights(q_lat, cache, block_table, query_start_loc, ctx, lse, scale, weights):
    """Add to ``weights [R, M]`` (fp32, in place, returned) what a step's attention gave every history row:

        weights[r, j] += sum over the tokens t of request r and the heads h of exp(scale * q_lat[t, h] . K[r, j] - lse[h, t])

    for ``j < min(ctx[t], M)``. ``cache`` is compact or bf16, ``block_table`` and ``weights`` are per request, ``query_start_loc``
    (int32 ``[R + 1]``) says which tokens are whose, ``ctx`` is per token. ``lse [16, T]`` is that of the whole softmax, which
    may cover more keys than the history (``s6_ops.merge_lse``); an infinite one marks an empty row and adds nothing. Sums are
    fp32 in a fixed order: the same call gives the same bits. Requests must have rows of ``weights`` of their own."""
    _same_device(cache, q_lat, block_table, query_start_loc, ctx, lse, weights)
    T, w = _query(q_lat)
    _, compact, page_stride, row_stride, block, num_blocks = _pages(cache, w)
    R = query_start_loc.shape[0] - 1
    qsl = _vector('query_start_loc', query_start_loc, R + 1)
    ctx = _vector('ctx', ctx, T)
    table_stride, cols, _ = _table(block_table, R)
    _rows2d('lse', lse, F32, (HEADS, T))
    weights_stride, M = _rows2d('weights', weights, F32)
    if weights.shape[0] != R:
        raise ValueError(f'weights has {weights.shape[0]} rows for {R} requests')
    lse = lse.contiguous()
    token_stride, head_stride, _ = q_lat.stride()
    shares, keys = account_shape(T, R, min(cols * block, M), _lib.device_cus(q_lat.get_device()), w)
    ws = torch.empty(shares * R * M, dtype=F32, device=weights.device) if shares > 1 else None
    _call('hla_s6_attention_weights', q_lat.device, q_lat.data_ptr(), T, HEADS, w, token_stride, head_stride,
          cache.data_ptr(), compact, page_stride, row_stride, block, num_blocks, block_table.data_ptr(), table_stride, cols,
          qsl.data_ptr(), R, ctx.data_ptr(), lse.data_ptr(), float(scale), weights.data_ptr(), weights_stride, M, keys, shares,
          _lib.ptr(ws), 0 if ws is None else ws.numel())
    return weights


def account_shape(num_tokens, num_reqs, rows, cu_count, width):
    """How ``attention_weights`` is cut: ``(shares of each request's tokens or 0, rows per workgroup)``. Steps of single
    tokens stream K past the queries (shares 0) in two workgroups a CU; longer ones hold K and stream the queries, the
    tokens shared out so that the last round of workgroups is a full one."""
    if num_tokens < 2 * num_reqs:
        per = -(-num_reqs * rows // (2 * cu_count))
        return 0, min(4096, max(128, -(-per // 128) * 128))
    groups = max(1, num_reqs * -(-rows // (256 if width <= 512 else 128)))
    slots, tokens = cu_count * (1 if width >= 512 else 2), num_tokens // max(1, num_reqs)
    # rounds of workgroups, each as long as a share's tokens and its rows' expansion (about 4 tokens' time); a reduction of
    # the shares costs about 4 as well
    cost = lambda z: -(-groups * z // slots) * (-(-tokens // z) + 4) + (4 if z > 1 else 0)
    return min(range(1, max(1, min(16, tokens // 4)) + 1), key=cost), 64


def select_rows(weights, positions, lengths, budget, protect_from):
    """Which rows of each request stay, and how they come together (an ``Eviction``; the inputs are left as they are).

    Of the first ``lengths[r]`` (int32 ``[R]``) rows the best ``budget`` (a number, or int32 ``[R]``) stay: first those whose
    ``positions[r, j]`` (int32 ``[R, M]``) is at least ``protect_from[r]`` (int32 ``[R]``), then by ``weights[r, j]`` (fp32 ``[R, M]``),
    descending; equal weights go to the earlier row, NaN ranks below everything. Rows that stay below the new length keep
    their place, and the i-th row behind it that stays moves to the i-th place left free: order among rows is not kept
    (attention over latent rows does not depend on it), positions tell it. ``move_rows`` applies the moves to a cache."""
    _same_device(weights, positions, lengths, protect_from, budget if torch.is_tensor(budget) else None)
    weights_stride, M = _rows2d('weights', weights, F32)
    R = weights.shape[0]
    positions_stride, _ = _rows2d('positions', positions, I32, (R, M))
    lengths = _vector('lengths', lengths, R)
    protect_from = _vector('protect_from', protect_from, R)
    budgets = None
    if torch.is_tensor(budget):
        budgets, budget = _vector('budget', budget, R), 0
    elif int(budget) < 0:
        raise ValueError(f'budget must not be negative, got {budget}')
    dev = weights.device
    e = Eviction(torch.empty(R, dtype=I32, device=dev), torch.empty(R, M, dtype=F32, device=dev),
                 torch.empty(R, M, dtype=I32, device=dev), torch.empty(R, M // 2, dtype=I32, device=dev),
                 torch.empty(R, M // 2, dtype=I32, device=dev))
    _call('hla_s6_select_rows', dev, weights.data_ptr(), weights_stride, positions.data_ptr(), positions_stride,
          lengths.data_ptr(), R, M, min(int(budget), 2 ** 31 - 1), _lib.ptr(budgets), protect_from.data_ptr(),
          *[t.data_ptr() for t in e])
    return e


def move_rows(cache, block_table, eviction):
    """Apply the row moves of ``select_rows`` to a cache (compact or bf16) in place, through the per-request
    ``block_table``. A request's pages must be its own: a page in two rows of the table would change for both. Moves through
    page ids outside the cache are skipped. The moves of a call run at once: in lists of a caller's own no source may be another
    move's target, nor a target named twice (``select_rows`` makes none such)."""
    source, target = eviction.source, eviction.target
    _same_device(cache, block_table, source, target)
    w, compact, page_stride, row_stride, block, num_blocks = _pages(cache)
    list_stride, count = _rows2d('source', source, I32)
    R = source.shape[0]
    if _rows2d('target', target, I32, (R, count))[0] != list_stride:
        source, target, list_stride = source.contiguous(), target.contiguous(), count
    table_stride, cols, _ = _table(block_table, R)
    _call('hla_s6_move_rows', cache.device, cache.data_ptr(), w, compact, page_stride, row_stride, block, num_blocks,
          block_table.data_ptr(), table_stride, cols, source.data_ptr(), target.data_ptr(), list_stride, count, R)
