"""Exact paged caches and the pages of any cache: their operators in plain form, and the calls a user makes of them.

An exact cache ``[pages, KV heads, block, 2d]`` holds the rows ``[K | V]`` of every KV head, in bf16 or in e4m3 times a scale per
head. The rows of request ``r`` lie in the pages of row ``r`` of a block table, ``block`` to a page. A pool of pages is
``tables [R, columns]`` (-1 behind a request's last page), ``lengths [R]`` (rows), ``refs [pages]`` (requests that hold a
page; 0: free) and ``free`` (a bit per page). Five operators:

* ``attn``: attention of a step's tokens over all their rows, or the last ``window`` of them (``exact_cache.attention``);
* ``store``: rows of new tokens into slots, -1 skipped (``exact_cache.store_rows``);
* ``fork``: samples of a prompt end, new ones begin on the prompt's pages and make room for a token: what they share and write
  to is copied (``release_requests``, ``fork_requests``, ``extend_requests``, ``copy_pages``);
* ``turn``: requests give back the pages behind a shorter length and take new ones up to a longer one (``release_requests``,
  ``extend_requests``);
* ``compact``: pages in use move to the front, the tables follow (``compact_pages``, ``copy_pages``).

Free pages are handed out lowest first, in the order of requests and of their columns.
"""
from __future__ import annotations

import importlib
import math
import random

import torch

own = False

PKG = 'hybrid-latent-attention_amd'
BF, F32, F64, I32, I64, E4 = (torch.bfloat16, torch.float32, torch.float64, torch.int32, torch.int64, torch.float8_e4m3fn)
TOP = 448.0     # the largest e4m3 value


def listed():
    return [
        # one interactive user on an exact layer of 16 heads: latency counts
        dict(name='attn_one', op='attn', tokens=1, ctx_min=993, ctx_max=993, kv_heads=16, group=1, dim=128, block=16, e4m3=False,
             window=0),
        # ordinary serving: grouped heads, requests of many lengths
        dict(name='attn_ragged', op='attn', tokens=32, ctx_min=1000, ctx_max=8160, kv_heads=8, group=4, dim=128, block=16,
             e4m3=False, window=0),
        # a full batch at 4K context, a KV head for every query head
        dict(name='attn_batch', op='attn', tokens=64, ctx_min=4096, ctx_max=4096, kv_heads=16, group=1, dim=128, block=16,
             e4m3=False, window=0),
        # two long documents in an 8-bit cache
        dict(name='attn_long', op='attn', tokens=2, ctx_min=100001, ctx_max=131000, kv_heads=8, group=8, dim=128, block=32,
             e4m3=True, window=0),
        # the rows of one decode step into an 8-bit cache; the rows of prompts
        dict(name='store_step', op='store', tokens=64, kv_heads=8, dim=128, block=16, e4m3=True),
        dict(name='store_prompts', op='store', tokens=8192, kv_heads=16, dim=128, block=16, e4m3=False),
        # four samples of one prompt; sixteen of each of sixteen prompts, on the caches of eight layers
        dict(name='fork_few', op='fork', prompts=1, samples=4, ctx_min=1000, ctx_max=1000, block=16, caches=2, width=512),
        dict(name='fork_groups', op='fork', prompts=16, samples=16, ctx_min=500, ctx_max=4090, block=16, caches=8, width=512),
        # a decode step's new rows; a full batch halves its histories and grows again
        dict(name='turn_step', op='turn', requests=64, ctx_min=1000, ctx_max=8160, shrink=1, block=16),
        dict(name='turn_evicted', op='turn', requests=256, ctx_min=8160, ctx_max=8160, shrink=4096, block=16),
        # holes that a few finished requests left; a large pool whose caches are to shrink
        dict(name='compact_few', op='compact', requests=8, ctx_min=500, ctx_max=1000, holes=0.2, block=16, caches=2, width=256),
        dict(name='compact_pool', op='compact', requests=64, ctx_min=2000, ctx_max=8160, holes=0.4, block=16, caches=4, width=512),
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, round(math.exp(rng.uniform(math.log(lo), math.log(hi))))))


def draw(rng):
    """One more case of the same kinds: sizes over the whole range, odd ones among them."""
    while True:
        op = rng.choices(('attn', 'store', 'fork', 'turn', 'compact'), (6, 2, 2, 2, 2))[0]
        case = dict(op=op, block=rng.choice((16, 16, 16, 32, 64, 24, 8)))
        lo, hi = sorted((_log_int(rng, 1, 8192), _log_int(rng, 1, 8192)))
        if op == 'attn':
            case.update(tokens=_log_int(rng, 1, 256), kv_heads=rng.choice((1, 2, 4, 8, 16)), dim=rng.choice((64, 128, 128, 256)),
                        group=rng.choice((1, 1, 2, 3, 4, 7, 8, 16)), e4m3=rng.random() < 0.4,
                        window=rng.choice((0, 0, 0, _log_int(rng, 1, 4096))))
            lo, hi = sorted((_log_int(rng, 1, 131000), _log_int(rng, 1, 131000)))
            case.update(ctx_min=rng.choice((lo, lo, lo, 0)), ctx_max=hi)
            if case['tokens'] * hi * case['kv_heads'] * max(1, case['group'] / 4) * case['dim'] <= 64 * 4096 * 16 * 128:
                return case
        elif op == 'store':
            case.update(tokens=_log_int(rng, 1, 8192), kv_heads=rng.choice((1, 2, 4, 8, 16)), dim=rng.choice((64, 128, 256)),
                        e4m3=rng.random() < 0.5)
            if case['tokens'] * case['kv_heads'] * case['dim'] <= 8192 * 16 * 128:
                return case
        elif op == 'fork':
            case.update(prompts=_log_int(rng, 1, 16), samples=_log_int(rng, 1, 16), ctx_min=lo, ctx_max=hi,
                        caches=rng.randint(1, 8), width=rng.choice((128, 256, 512)))
            if case['prompts'] * hi * case['caches'] * case['width'] <= 16 * 4090 * 8 * 512:
                return case
        elif op == 'turn':
            case.update(requests=_log_int(rng, 1, 256), ctx_min=lo, ctx_max=hi, shrink=_log_int(rng, 1, hi))
            return case
        else:
            case.update(requests=_log_int(rng, 1, 64), ctx_min=lo, ctx_max=hi, holes=round(rng.uniform(0.05, 0.6), 2),
                        caches=rng.randint(1, 6), width=rng.choice((128, 256, 512)))
            if case['requests'] * hi * case['caches'] * case['width'] <= 64 * 5080 * 4 * 512:
                return case


# ---- sizes -----------------------------------------------------------------------------------------------------------

def _lengths(case, count):
    """Rows per request, the same for every seed (a case's work is fixed); one at the largest."""
    rng = random.Random(f"{count} {case['ctx_min']} {case['ctx_max']}")
    n = [rng.randint(case['ctx_min'], case['ctx_max']) for _ in range(count)]
    n[0] = case['ctx_max']
    return n


def _pages(case, rows):
    return -(-rows // case['block'])


def _shrunk(case, n):
    """Lengths after the rows behind have gone; one request of nine has finished."""
    return [0 if r % 9 == 4 else max(1, x - case['shrink']) for r, x in enumerate(n)]


def _page_bytes(case):
    return case['caches'] * case['block'] * 2 * case['width'] * 2


def work(case):
    op = case['op']
    if op == 'attn':
        n = [min(x, case['window'] or x) for x in _lengths(case, case['tokens'])]
        kv, q = case['kv_heads'] * case['dim'] * 2, case['kv_heads'] * case['group'] * case['dim']
        return dict(bytes=sum(n) * kv * (1 if case['e4m3'] else 2) + case['tokens'] * q * 4, flops=sum(n) * q * 4)
    if op == 'store':
        values = case['tokens'] * case['kv_heads'] * case['dim'] * 2
        return dict(bytes=values * (3 if case['e4m3'] else 4) + case['tokens'] * 8, flops=values)
    if op == 'fork':
        n = _lengths(case, case['prompts'])
        shared, copied = sum(_pages(case, x) for x in n), sum(x % case['block'] > 0 for x in n)
        # a child's entries are dropped and written, the counts of their pages changed twice; its last page is copied
        return dict(bytes=case['samples'] * (24 * shared + 2 * copied * _page_bytes(case)), flops=case['samples'] * 4 * shared)
    if op == 'turn':
        n = _lengths(case, case['requests'])
        moved = sum(_pages(case, x) - _pages(case, y) for x, y in zip(n, _shrunk(case, n)))
        return dict(bytes=16 * case['requests'] + 24 * moved, flops=4 * (moved + case['requests']))
    used = sum(_pages(case, x) for x in _lengths(case, case['requests']))
    moved = round(used * case['holes'] / (1 + case['holes']))    # the share of the used pages that lies behind them
    return dict(bytes=8 * used + 2 * moved * _page_bytes(case), flops=4 * used)


# ---- inputs ----------------------------------------------------------------------------------------------------------

def _noise(gen, *shape):
    return torch.randn(*shape, generator=gen, device='cuda')


def _scales(gen, heads):
    """A scale per head of an e4m3 cache, as a calibration leaves them."""
    return torch.exp(0.3 * _noise(gen, heads)) / 64


def _rows(gen, case, rows):
    """``[rows, KV heads, d]`` of keys or values: channels and heads of different sizes."""
    h, d = case['kv_heads'], case['dim']
    return (_noise(gen, rows, h, d) * torch.exp(0.3 * _noise(gen, h, d))).to(BF)


def _to_e4m3(x, scale):
    return (x.float() / scale[:, None]).clamp(-TOP, TOP).to(E4)


def _pool(gen, case, lengths, pages, shared=None):
    """A pool whose requests' pages lie in random order. ``shared``: the request whose pages request r has instead of its own."""
    n = torch.tensor(lengths, dtype=I32, device='cuda')
    cols = _pages(case, max(lengths) + 1)
    held = (n + case['block'] - 1) // case['block']
    own_pages = held if shared is None else torch.where(shared == torch.arange(len(lengths), device='cuda'), held, 0)
    seen = torch.arange(cols, device='cuda') < own_pages[:, None]
    tables = torch.full((len(lengths), cols), -1, dtype=I32, device='cuda')
    tables[seen] = torch.randperm(pages, generator=gen, device='cuda')[:int(own_pages.sum())].to(I32)
    if shared is not None:
        tables = tables[shared]
    refs = torch.bincount(tables[tables >= 0].long(), minlength=pages).to(I32)
    bits = torch.zeros(-(-pages // 32) * 32, dtype=I64, device='cuda')
    bits[:pages] = (refs == 0).long()
    words = (bits.view(-1, 32) << torch.arange(32, device='cuda')).sum(-1)
    return dict(tables=tables, lengths=n, refs=refs, free=torch.where(words >> 31 > 0, words - (1 << 32), words).to(I32))


def _caches(gen, case, pages):
    return [_noise(gen, pages, 1, case['block'], 2 * case['width']).to(BF) for _ in range(case['caches'])]


def prepare(case, seed):
    gen = torch.Generator(device='cuda').manual_seed(seed)
    op, block = case['op'], case['block']
    s = dict(case)
    if op == 'attn':
        T, h, d, n = case['tokens'], case['kv_heads'], case['dim'], _lengths(case, case['tokens'])
        pages = sum(_pages(case, x) for x in n) + 1
        pool = _pool(gen, case, n, pages)
        s.update(table=pool['tables'].clamp(min=0), ctx=pool['lengths'], max_rows=max(n), scale=d ** -0.5)
        # pages with the rows of all heads one behind the other; what lies outside the requests' rows is not to be read
        cache = torch.full((pages, block, h, 2 * d), float('nan'), dtype=BF, device='cuda')
        at = torch.arange(pool['tables'].shape[1] * block, device='cuda')
        seen = at < pool['lengths'][:, None]
        slots = (pool['tables'].long().repeat_interleave(block, 1) * block + at % block)[seen]
        size = torch.exp(0.3 * _noise(gen, h, 2 * d))
        flat = cache.view(-1, h, 2 * d)
        for part in slots.split(max(1, (1 << 26) // (h * d))):
            flat[part] = (_noise(gen, part.shape[0], h, 2 * d) * size).to(BF)
        if case['e4m3']:
            s.update(k_scale=_scales(gen, h), v_scale=_scales(gen, h))
            both = torch.cat((s['k_scale'][:, None].expand(h, d), s['v_scale'][:, None].expand(h, d)), 1)
            out = torch.empty_like(cache, dtype=E4)
            step = max(1, (1 << 26) // (block * h * d))
            for i in range(0, pages, step):
                out[i:i + step] = (cache[i:i + step].float() / both).clamp(-TOP, TOP).to(E4)
            cache = out
        s['cache'] = cache.transpose(1, 2)      # [pages, KV heads, block, 2d]
        s['q'] = _noise(gen, T, h * case['group'], d).to(BF)
        return s
    if op == 'store':
        T, h, d = case['tokens'], case['kv_heads'], case['dim']
        pages = _pages(case, 2 * T) + 1
        s.update(key=_rows(gen, case, T), value=_rows(gen, case, T))
        s['slots'] = torch.randperm(pages * block, generator=gen, device='cuda')[:T]
        s['slots'][torch.rand(T, generator=gen, device='cuda') < 0.02] = -1     # padding
        cache = _noise(gen, pages, block, h, 2 * d).to(BF)
        if case['e4m3']:
            s.update(k_scale=_scales(gen, h), v_scale=_scales(gen, h))
            cache = cache.to(E4)
        s['cache'] = cache.transpose(1, 2)
        return s
    if op == 'fork':
        P, S = case['prompts'], case['samples']
        n = _lengths(case, P)
        pages = sum(_pages(case, x) for x in n) + 2 * P * S + 8
        # the samples of before hold their prompts' pages and, once they have written, one of their own
        shared = torch.arange(P * (1 + S), device='cuda')
        shared[P:] = torch.arange(P * S, device='cuda') % P
        s.update(_pool(gen, case, n + n * S, pages, shared), caches=_caches(gen, case, pages))
        order = torch.randperm(P * S, generator=gen, device='cuda')
        s['children'] = (P + order).to(I32)
        s['parents'] = (order % P).to(I32)
        s['target'] = s['lengths'] + (shared != torch.arange(P * (1 + S), device='cuda')).to(I32)
        return s
    if op == 'turn':
        n = _lengths(case, case['requests'])
        s.update(_pool(gen, case, n, math.ceil(1.1 * sum(_pages(case, x) for x in n)) + 3))
        s['requests'] = torch.randperm(len(n), generator=gen, device='cuda').to(I32)
        s['shorter'] = torch.tensor(_shrunk(case, n), dtype=I32, device='cuda')[s['requests'].long()]
        s['target'] = s['lengths'].clone()
        return s
    n = _lengths(case, case['requests'])
    pages = math.ceil((1 + case['holes']) * sum(_pages(case, x) for x in n))
    pool = _pool(gen, case, n, pages)
    s.update({k + '0': v for k, v in pool.items()}, caches=_caches(gen, case, pages))
    return s


# ---- one pass --------------------------------------------------------------------------------------------------------

def run(s):
    if own:
        amd = importlib.import_module(PKG)
        ec, pg = amd.exact_cache, amd.pages
        if s['op'] == 'attn':
            return ec.attention(s['q'], s['cache'], s['table'], s['ctx'], s['scale'], s['max_rows'], window=s['window'],
                                k_scale=s.get('k_scale'), v_scale=s.get('v_scale'))
        if s['op'] == 'store':
            ec.store_rows(s['key'], s['value'], s['slots'], s['cache'], s.get('k_scale'), s.get('v_scale'))
            return s['cache']
        if s['op'] == 'compact':
            # (its holes are gone afterwards: every pass compacts a copy of the pool)
            pool = pg.Pool(s['tables0'].clone(), s['lengths0'], s['refs0'].clone(), s['free0'].clone(), s['block'])
            moves = pg.compact_pages(pool)
            pg.copy_pages(s['caches'], moves.source, moves.target)
            return [pool.tables, pool.refs, moves.source, moves.target, s['caches']]
        pool = pg.Pool(s['tables'], s['lengths'], s['refs'], s['free'], s['block'])
        if s['op'] == 'turn':
            pg.release_requests(pool, s['requests'], s['shorter'])
            e = pg.extend_requests(pool, s['target'])
            return [pool.tables, pool.lengths, pool.refs, e.ok]
        pg.release_requests(pool, s['children'])
        ok = pg.fork_requests(pool, s['parents'], s['children'])
        e = pg.extend_requests(pool, s['target'])
        pg.copy_pages(s['caches'], e.source, e.target)
        return [pool.tables, pool.lengths, pool.refs, ok, e.ok, e.source, e.target, s['caches']]
    if s['op'] == 'attn':
        return _attention(s)
    if s['op'] == 'store':
        _store(s)
        return s['cache']
    if s['op'] == 'compact':
        tables, refs, source, target = _compact(s)
        _copy(s['caches'], source, target)
        return [tables, refs, source, target, s['caches']]
    if s['op'] == 'turn':
        _release(s, s['requests'], s['shorter'])
        ok, _, _ = _extend(s)
        return [s['tables'], s['lengths'], s['refs'], ok]
    _release(s, s['children'], torch.zeros_like(s['children']))
    forked = _fork(s)
    ok, source, target = _extend(s)
    _copy(s['caches'], source, target)
    return [s['tables'], s['lengths'], s['refs'], forked, ok, source, target, s['caches']]


def _attention(s):
    """Output (bf16) and log-sum-exp over the gathered rows, all tokens at once."""
    q, cache, ctx = s['q'], s['cache'], s['ctx'].long()
    T, H, d = q.shape
    h, block = cache.shape[1], s['block']
    rows = cache.transpose(1, 2)[s['table'].long()].flatten(1, 2)[:, :s['max_rows']].transpose(1, 2)    # [T, h, rows, 2d]
    at = torch.arange(rows.shape[2], device='cuda')
    seen = (at < ctx[:, None]) & (at >= ctx[:, None] - (s['window'] or 1 << 30))
    k = torch.where(seen[:, None, :, None], rows[..., :d].float(), 0)
    score = torch.matmul(q.float().view(T, h, H // h, d), k.transpose(2, 3).contiguous()) * s['scale']
    if s['e4m3']:
        score = score * s['k_scale'].float()[:, None, None]
    score = torch.where(seen[:, None, None], score, -math.inf)
    del k
    top = score.amax(-1, keepdim=True).clamp(min=-1e30)
    p = torch.exp(score - top)
    total = p.sum(-1, keepdim=True)
    v = torch.where(seen[:, None, :, None], rows[..., d:].float(), 0)
    o = torch.where(total > 0, torch.matmul(p, v) / total, 0)
    if s['e4m3']:
        o = o * s['v_scale'].float()[:, None, None]
    lse = (top + torch.log(total)).view(T, H).t().contiguous()
    return o.reshape(T, H, d).to(BF), lse


def _store(s):
    keep = s['slots'] >= 0
    slots, d = s['slots'][keep], s['dim']
    flat = s['cache'].transpose(1, 2).view(-1, s['kv_heads'], 2 * d)
    for at, rows, scale in ((0, s['key'], s.get('k_scale')), (d, s['value'], s.get('v_scale'))):
        part = rows[keep]
        flat[:, :, at:at + d][slots] = part if scale is None else _to_e4m3(part, scale)


def _held(s):
    """Which entries of the tables hold a page."""
    n = (s['lengths'] + s['block'] - 1) // s['block']
    return torch.arange(s['tables'].shape[1], device='cuda') < n[:, None]


def _count(s, tables, held, by):
    s['refs'].index_add_(0, tables[held].long(), torch.full((int(held.sum()),), by, dtype=I32, device='cuda'))


def _release(s, requests, lengths):
    """Pages behind the shorter lengths of the requests."""
    before, rows = _held(s), requests.long()
    s['lengths'][rows] = torch.minimum(s['lengths'][rows], lengths)
    gone = before & ~_held(s)
    _count(s, s['tables'], gone, -1)
    s['tables'][gone] = -1


def _fork(s):
    """Children (without rows, each named once) take over the pages of parents that are no children."""
    parents, children = s['parents'].long(), s['children'].long()
    ok = s['lengths'][children] == 0
    s['lengths'][children] = s['lengths'][parents]
    s['tables'][children] = s['tables'][parents]
    new = torch.zeros_like(s['lengths'], dtype=torch.bool)
    new[children] = True
    _count(s, s['tables'], _held(s) & new[:, None], 1)
    return ok


def _extend(s):
    """Room for the rows up to ``target``: new pages behind the last, a copy of a last page that others hold too."""
    tables, refs, block = s['tables'], s['refs'], s['block']
    R, cols = tables.shape
    held = _held(s)
    target = torch.maximum(s['target'], s['lengths'])
    col = torch.arange(cols, device='cuda')
    grows = target > s['lengths']
    new = (col < ((target + block - 1) // block)[:, None]) & ~held
    copied = held & (grows[:, None] & (col >= (s['lengths'] // block)[:, None])) & (refs[tables.clamp(min=0).long()] > 1)
    want = new | copied
    free = (refs == 0).nonzero()[:, 0]
    demand = want.sum(1)
    ok = (demand == 0) | (demand.cumsum(0) <= free.shape[0])
    want, copied = want & ok[:, None], copied & ok[:, None]
    ids = free[:int(want.sum())].to(I32)
    last = copied.any(1)
    source = torch.where(last, torch.where(copied, tables, 0).sum(1).to(I32), -1)
    _count(s, tables, copied, -1)
    tables[want] = ids
    refs[ids.long()] = 1
    s['lengths'].copy_(torch.where(ok, target, s['lengths']))
    return ok, source, torch.where(last, torch.where(copied, tables, 0).sum(1).to(I32), -1)


def _compact(s):
    """Tables and counts with the pages in use at the front, and the moves that bring them there."""
    tables, refs = s['tables0'], s['refs0'].clone()
    N = refs.shape[0]
    used = int((refs > 0).sum())
    movers, holes = (refs[used:] > 0).nonzero()[:, 0] + used, (refs[:used] == 0).nonzero()[:, 0]
    place = torch.arange(N, device='cuda')
    place[movers] = holes
    refs[holes] = refs[movers]
    refs[movers] = 0
    lists = torch.full((2, N // 2), -1, dtype=I32, device='cuda')
    lists[0, :movers.shape[0]] = movers.to(I32)
    lists[1, :holes.shape[0]] = holes.to(I32)
    return torch.where(tables >= 0, place[tables.clamp(min=0).long()].to(I32), tables), refs, lists[0], lists[1]


def _copy(caches, source, target):
    moves = source >= 0
    a, b = source[moves].long(), target[moves].long()
    for cache in caches:
        cache[b] = cache[a]


# ---- in 64 bits ------------------------------------------------------------------------------------------------------

def exact(case, seed):
    """What attention and stores give in 64 bits, from the definition; of pools the caches (the rest is whole numbers)."""
    if case['op'] == 'turn':
        return None
    s = prepare(case, seed)
    if case['op'] in ('fork', 'compact'):
        return _exact_caches(s)
    if case['op'] == 'store':
        return _exact_store(s)
    h, d, G, block = case['kv_heads'], case['dim'], case['group'], case['block']
    outs, lses = [], []
    for t, n in enumerate(s['ctx'].tolist()):
        first = max(0, n - case['window']) if case['window'] else 0
        rows = torch.arange(first, n, device='cuda')
        kv = s['cache'][s['table'][t].long()[rows // block], :, rows % block].to(F64)      # [rows, h, 2d]
        if case['e4m3']:
            kv = kv * torch.cat((s['k_scale'][:, None].expand(h, d), s['v_scale'][:, None].expand(h, d)), 1).to(F64)
        q = s['q'][t].to(F64).view(h, G, d)
        score = torch.einsum('hgd,nhd->hgn', q, kv[..., :d]) * s['scale']
        lse = torch.logsumexp(score, -1)
        outs.append(torch.einsum('hgn,nhd->hgd', torch.exp(score - lse[..., None]), kv[..., d:]).reshape(h * G, d))
        lses.append(lse.reshape(-1))
    return torch.stack(outs), torch.stack(lses, 1)


def _exact_store(s):
    """Every value by hand: the nearest multiple of the step of its binade, ties to the even one, at most 448."""
    cache, block, d = s['cache'].to(F64).clone(), s['block'], s['dim']
    keep = (s['slots'] >= 0).nonzero()[:, 0]
    page, row = s['slots'][keep] // block, s['slots'][keep] % block
    for at, rows, scale in ((0, s['key'], s.get('k_scale')), (d, s['value'], s.get('v_scale'))):
        x = rows[keep].to(F64)
        if scale is not None:
            x = (x / scale.to(F64)[:, None]).clamp(-TOP, TOP)
            step = torch.exp2(torch.floor(torch.log2(x.abs().clamp(min=2.0 ** -6))) - 3)
            x = torch.round(x / step) * step
        cache[page, :, row, at:at + d] = x
    return cache


def _exact_caches(s):
    """Page by page: whose copy it is afterwards."""
    caches = [c.to(F64) for c in s['caches']]
    if s['op'] == 'compact':
        refs = s['refs0'].tolist()
        used = sum(x > 0 for x in refs)
        pairs = zip((p for p in range(used, len(refs)) if refs[p]), (p for p in range(used) if not refs[p]))
        other = 4
    else:
        P, block = s['prompts'], s['block']
        tables, n = s['tables'][:P].tolist(), s['lengths'][:P].tolist()
        held = {p for t, x in zip(tables, n) for p in t[:_pages(s, x)]}
        free = (p for p in range(caches[0].shape[0]) if p not in held)
        taken = [(j % P, next(free)) for j in range(P * s['samples'])]      # a page for every sample, in the order of rows
        pairs = ((tables[r][n[r] // block], p) for r, p in taken if n[r] % block)
        other = 7
    pairs = list(pairs)
    if pairs:
        source, target = torch.tensor(pairs, device='cuda').t()
        for c in caches:
            c[target] = c[source]
    return [None] * other + [caches]
