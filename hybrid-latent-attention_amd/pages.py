"""Pools of cache pages on MI355X: requests that share, take and drop pages, and caches that shrink.

A pool says which pages of a cache, or of any number of caches with common block tables, belong to whom; its tables and lengths
are what the attention, store and eviction operators take. ``fork_requests`` lets requests share the pages of another (the samples
of one prompt), ``extend_requests`` makes room for rows that are about to be written, ``release_requests`` gives pages back (of a
finished request, or behind the length that an eviction left), ``compact_pages`` moves the pages in use to the front of the
cache. None of them touches a cache: where pages have to be copied they return the pairs, and ``copy_pages`` copies them, one call
for every cache geometry.

A row is written after ``extend_requests`` has made room for it: then its page belongs to its request alone. Rows that are moved
(``compact_cache.move_rows``) need the pages of all rows to be their request's own: ``extend_requests(pool, pool.lengths,
write_from=zeros)``.

All results are functions of the pool and the arguments: free pages are handed out lowest first, in the order of requests and of
their columns. Everything is enqueued on the current stream of the pool's device, nothing synchronised, every call capturable
in a HIP graph; calls on one pool must not overlap. Checks and errors are those of ``compact_cache``.
"""
from __future__ import annotations

import ctypes
from collections import namedtuple

import torch

from . import _lib
from .compact_cache import _call, _rows2d, _same_device, _vector

I32 = torch.int32
MAX_REQUESTS = 8192

#: What ``extend_requests`` returns: ``ok [R]`` (bool), and the pages to copy.
Extension = namedtuple('Extension', 'ok source target')
#: Pages to copy: int32 lists, -1 where there is nothing to do.
Moves = namedtuple('Moves', 'source target')


class Pool:
    """The state of a pool, int32 tensors on one device: ``tables [R, C]`` (any row stride), the pages of request ``r``, -1 behind its
    last; ``lengths [R]``, its rows; ``refs [N]``, the requests that hold a page; ``free [ceil(N / 32)]``, bit ``p % 32`` of word ``p //
    32`` set where ``refs[p]`` is 0; and ``block``, the rows per page. Checked here, once; the operators below write into the tensors,
    which cannot be exchanged for others."""

    __slots__ = ('tables', 'lengths', 'refs', 'free', 'block', '_args')

    def __init__(self, tables, lengths, refs, free, block):
        stride, cols = _rows2d('tables', tables, I32)
        R, N, block = tables.shape[0], refs.shape[0], int(block)
        if R > MAX_REQUESTS or block < 1:
            raise ValueError(f'no pool for {R} requests (at most {MAX_REQUESTS}) with pages of {block} rows')
        for name, t, n in (('lengths', lengths, R), ('refs', refs, N), ('free', free, -(-N // 32))):
            if _vector(name, t, n) is not t:
                raise ValueError(f'{name} must be contiguous')
            if t.device != tables.device:
                raise RuntimeError(f'tensors on {tables.device} and {t.device}')
        args = (tables.data_ptr(), stride, R, cols, lengths.data_ptr(), refs.data_ptr(), N, free.data_ptr(), block)
        for name, value in zip(self.__slots__, (tables, lengths, refs, free, block, args)):
            object.__setattr__(self, name, value)

    def __setattr__(self, name, value):
        raise AttributeError(f'{name} of a pool is written into, not exchanged')

    def __reduce__(self):
        return Pool, (self.tables, self.lengths, self.refs, self.free, self.block)


def new_pool(num_pages, block, max_requests, max_rows, device, reserved=0):
    """A pool of ``num_pages`` free pages of ``block`` rows for ``max_requests`` requests of at most ``max_rows`` rows. The first
    ``reserved`` pages belong to nobody and are never handed out."""
    num_pages, block, max_requests, max_rows, reserved = (int(x) for x in (num_pages, block, max_requests, max_rows, reserved))
    if block < 1 or not 0 <= reserved <= num_pages or not 0 <= max_requests <= MAX_REQUESTS or max_rows < 0:
        raise ValueError(f'no pool of {num_pages} pages ({reserved} reserved) of {block} rows for {max_requests} requests '
                         f'(at most {MAX_REQUESTS}) of {max_rows} rows')
    refs = torch.zeros(num_pages, dtype=I32, device=device)
    refs[:reserved] = 1
    bits = torch.zeros(-(-num_pages // 32) * 32, dtype=torch.int64, device=device)
    bits[reserved:num_pages] = 1
    words = (bits.view(-1, 32) << torch.arange(32, device=device)).sum(-1)
    return Pool(torch.full((max_requests, -(-max_rows // block)), -1, dtype=I32, device=device),
                torch.zeros(max_requests, dtype=I32, device=device), refs,
                torch.where(words >> 31 > 0, words - (1 << 32), words).to(I32), block)


def _apart(pool, vector, in_place):
    """``vector``, or a copy of it where it lies on the pool's lengths, which change while requests are worked on; the lengths
    themselves are fine where a request reads no entry but its own (``in_place``)."""
    offset, held = vector.data_ptr() - pool._args[4], pool.lengths.shape[0]
    if -4 * vector.shape[0] < offset < 4 * held and not (in_place and offset == 0):
        return vector.clone()
    return vector


def release_requests(pool, requests, lengths=None):
    """Requests ``requests`` (int32 ``[n]``) keep their first ``lengths[i]`` rows (int32 ``[n]``; none without it; more than a request
    has: all) and give back the pages behind them; a page is free once nobody holds it. Numbers outside the pool are skipped; of a
    request named twice the shorter length holds."""
    n = requests.shape[0]
    _same_device(pool.tables, requests, lengths)
    requests = _vector('requests', requests, n)
    if lengths is not None:
        lengths = _apart(pool, _vector('lengths', lengths, n), False)
    _call('hla_s6_pool_release', pool.tables.device, *pool._args, requests.data_ptr(), _lib.ptr(lengths), n)


def fork_requests(pool, parents, children):
    """Requests ``children`` (int32 ``[n]``, without rows) take over the pages and lengths of ``parents`` (int32 ``[n]``); pages are
    shared, nothing is copied. Returns ``ok [n]`` (bool): False, and nothing done, where a number is outside the pool, the child
    has rows or was named before in the list, or the parent is itself among the children."""
    n = parents.shape[0]
    _same_device(pool.tables, parents, children)
    parents, children = _vector('parents', parents, n), _vector('children', children, n)
    ok = torch.empty(n, dtype=torch.bool, device=pool.tables.device)
    _call('hla_s6_pool_fork', ok.device, *pool._args, parents.data_ptr(), children.data_ptr(), n, ok.data_ptr())
    return ok


def extend_requests(pool, lengths, write_from=None):
    """Room for the rows ``write_from[r] .. lengths[r]`` of every request (int32 ``[R]`` each; ``write_from`` defaults to the pool's
    lengths: the rows to come), whose length becomes ``lengths[r]`` (it stays where it is longer already). Columns behind a
    request's last page get free pages. Columns with rows to write whose page others hold too get a free page in its place, and the
    pairs ``(source, target)`` of the returned ``Extension`` say what to copy (``copy_pages``) before the rows are written.

    ``ok[r]`` is False, and the request as it was, where ``lengths[r]`` does not fit the table or it and the requests before it ask for
    more pages than are free: no request overtakes one that waits. (Requests that share a page and write to it in the same call get a
    copy each.) The lists are ``[R]``, or with ``write_from`` ``[R, C]``, an entry per entry of the table."""
    _same_device(pool.tables, lengths, write_from)
    tables = pool.tables
    R, C = tables.shape
    lengths = _apart(pool, _vector('lengths', lengths, R), True)
    if write_from is not None:
        write_from = _apart(pool, _vector('write_from', write_from, R), True)
    dev = tables.device
    ok = torch.empty(R, dtype=torch.bool, device=dev)
    shape = (R,) if write_from is None else (R, C)
    source, target = torch.empty(shape, dtype=I32, device=dev), torch.empty(shape, dtype=I32, device=dev)
    scratch = None if write_from is None else torch.empty(R * (C + 1), dtype=I32, device=dev)
    _call('hla_s6_pool_extend', dev, *pool._args, lengths.data_ptr(), _lib.ptr(write_from), ok.data_ptr(), source.data_ptr(),
          target.data_ptr(), _lib.ptr(scratch))
    return Extension(ok, source, target)


def compact_pages(pool):
    """Pages in use move to the front: with ``U`` of them, the i-th page in use at or behind ``U`` takes the i-th free place before it,
    in the tables and counts. The returned ``Moves`` (int32 ``[N // 2]``, -1 behind the last) are to be copied in every cache of the
    pool before anything reads it; pages from ``U`` on are free then. Holders that no table knows find their pages by the moves."""
    _same_device(pool.tables)
    dev, N = pool.refs.device, pool.refs.shape[0]
    source, target = torch.empty(N // 2, dtype=I32, device=dev), torch.empty(N // 2, dtype=I32, device=dev)
    scratch = torch.empty(N + 2, dtype=I32, device=dev)
    _call('hla_s6_pool_compact', dev, *pool._args, source.data_ptr(), target.data_ptr(), scratch.data_ptr())
    return Moves(source, target)


def copy_pages(caches, source, target):
    """Page ``target[i]`` of every cache becomes a copy of its page ``source[i]`` (int32 lists of one shape; pairs with a number
    outside the cache, as -1, are skipped). ``caches`` is a tensor or a sequence of tensors of one shape, type and strides whose
    first dimension is the page, each page a dense piece of memory (bf16, compact and exact caches are). The copies run at once: no
    source may be another pair's target, nor a target named twice (the operators of this module make none such)."""
    caches = [caches] if torch.is_tensor(caches) else list(caches)
    if not caches:
        return
    first = caches[0]
    shape, stride, dtype = first.shape, first.stride(), first.dtype
    for c in caches[1:]:
        if c.shape != shape or c.stride() != stride or c.dtype != dtype:
            raise ValueError('the caches of a call must have one shape, type and strides')
    _same_device(*caches, source, target)
    size = 1
    for s, n in sorted(zip(stride[1:], shape[1:])):
        if n > 1 and s != size:
            raise ValueError(f'the pages of a cache must be dense, got strides {stride} of {tuple(shape)}')
        size *= n
    if not len(shape) or (shape[0] > 1 and stride[0] < size):
        raise ValueError(f'caches are [num_blocks, ...] with pages apart, got strides {stride} of {tuple(shape)}')
    if source.shape != target.shape or source.dtype != I32 or target.dtype != I32:
        raise ValueError(f'source and target must be int32 lists of one shape, got {source.dtype} {tuple(source.shape)} and '
                         f'{target.dtype} {tuple(target.shape)}')
    source, target = source.contiguous(), target.contiguous()
    width = first.element_size()
    pointers = (ctypes.c_void_p * len(caches))(*[c.data_ptr() for c in caches])
    _call('hla_s6_copy_pages', first.device, pointers, len(caches), stride[0] * width, size * width, shape[0],
          source.data_ptr(), target.data_ptr(), source.numel())
