"""Whole exact caches on the GPU against 64-bit forms.

Tolerances. The output is rounded to bf16 (half a step: 2^-8 relative); a weight goes into its product as its upper bf16 half and the
rest, below 2^-7 of it, rounded to bf16 (2^-8 of the rest): 2^-15 sum p |v|. fp32 scores are off by at most (d + 2) 2^-24 scale sum
|q k| =: e (products of bf16 and of e4m3 values are exact, a scale of the cache is one more rounding), which moves a weight by a
factor of up to exp(2 e); exponentials and sums add 2^-20 of the sum at the sizes here (2^-22 per exponential and per factor between
parts, sums of up to 2^13 terms in chains of at most 2^5 per lane and part). The log-sum-exp is off by e, those sums and its own
rounding."""
import math

import numpy as np
import pytest
import torch

from s6util import dev_i32, dev_i64

pytestmark = pytest.mark.gpu
HALF = 2.0 ** -8
E4 = torch.float8_e4m3fn


@pytest.fixture(scope='module')
def ec(pkg):
    return pkg.exact_cache


class Cache:
    """Requests of given lengths in pages in random order; everything outside their rows is NaN."""

    def __init__(self, seed, lengths, kv_heads, d, block=16, e4m3=False, heads_first=False, extra_cols=1):
        g = torch.Generator(device='cuda').manual_seed(seed)
        self.n, self.h, self.d, self.block, self.e4m3 = list(lengths), kv_heads, d, block, e4m3
        cols = max(1, -(-max(self.n) // block)) + extra_cols
        pages = len(self.n) * cols + 2
        self.table = (torch.randperm(pages - 2, generator=g, device='cuda') + 2)[:len(self.n) * cols].view(-1, cols).to(torch.int32)
        noise = lambda *s: torch.randn(*s, generator=g, device='cuda')
        self.rows = [noise(n, kv_heads, 2 * d) * torch.exp(0.3 * noise(kv_heads, 2 * d)) for n in self.n]
        shape = (pages, kv_heads, block, 2 * d) if heads_first else (pages, block, kv_heads, 2 * d)
        self.cache = torch.full(shape, math.nan, device='cuda').to(E4 if e4m3 else torch.bfloat16)
        if not heads_first:
            self.cache = self.cache.transpose(1, 2)
        self.k_scale = self.v_scale = None
        if e4m3:
            self.k_scale, self.v_scale = torch.exp(noise(kv_heads)) / 64, torch.exp(noise(kv_heads)) / 64
        for r, rows in enumerate(self.rows):
            at = torch.arange(rows.shape[0], device='cuda')
            held = rows.clamp(-440, 440).to(self.cache.dtype)
            raw = self.cache.view(torch.uint8) if e4m3 else self.cache
            raw[self.table[r].long()[at // block], :, at % block] = held.view(torch.uint8) if e4m3 else held
            rows = held.double()
            if e4m3:
                rows[..., :d] *= self.k_scale.double()[:, None]
                rows[..., d:] *= self.v_scale.double()[:, None]
            self.rows[r] = rows


def query(seed, T, H, d, size=1.0):
    g = torch.Generator(device='cuda').manual_seed(seed)
    return (size * torch.randn(T, H, d, generator=g, device='cuda')).to(torch.bfloat16)


def check(o, lse, q, cache, requests, ctx, scale, window=0):
    """Every token against float64, with the bounds above."""
    T, H, d = q.shape
    G = H // cache.h
    assert o.shape == q.shape and o.dtype == torch.bfloat16 and lse.shape == (H, T) and lse.dtype == torch.float32
    for t, n in enumerate(ctx):
        rows = cache.rows[requests[t]][max(0, n - window) if window else 0:max(n, 0)]
        if not rows.shape[0]:
            assert (o[t] == 0).all() and torch.isneginf(lse[:, t]).all(), (t, n)
            continue
        k, v = rows[..., :d].repeat_interleave(G, 1), rows[..., d:].repeat_interleave(G, 1)      # [n, H, d]
        x = q[t].double()
        s = (x * k).sum(-1) * scale
        want_lse = torch.logsumexp(s, 0)
        p = torch.exp(s - want_lse)[..., None]
        want, size = (p * v).sum(0), (p * v.abs()).sum(0)
        e = (d + 2) * 2.0 ** -24 * scale * (x.abs() * k.abs()).sum(-1).amax(0)
        bound = 1.001 * HALF * want.abs() + (2.0 ** -15 + torch.expm1(2 * e) + 2.0 ** -20)[:, None] * size * 1.01
        off = (o[t].double() - want).abs()
        assert (off <= bound).all(), (t, n, float((off - bound).max()), float((off / bound).max()))
        off = (lse[:, t].double() - want_lse).abs()
        assert (off <= e + 2.0 ** -20 + 2.0 ** -22 * want_lse.abs()).all(), (t, n, float(off.max()))


def attend(ec, q, c, ctx, scale=None, **more):
    """Attention of token t over request t."""
    scale = q.shape[-1] ** -0.5 if scale is None else scale
    return ec.attention(q, c.cache, c.table, dev_i32(np.array(ctx)), scale, max(max(ctx), 0), k_scale=c.k_scale, v_scale=c.v_scale,
                        **more)


# ---- attention ---------------------------------------------------------------------------------------------------------

@pytest.mark.parametrize('e4m3', [False, True])
@pytest.mark.parametrize('d', [64, 128, 256])
@pytest.mark.parametrize('kv_heads,G,block', [(16, 1, 16), (8, 4, 16), (2, 7, 48), (1, 16, 24), (3, 1, 1), (2, 17, 16), (1, 40, 5)])
def test_attention(ec, kv_heads, G, block, d, e4m3):
    n = [1, 0, 15, 16, 17, 33, 257, 64, 1000, 129]
    c = Cache(d + G, n, kv_heads, d, block, e4m3, heads_first=G == 7)
    q = query(d * G, len(n), kv_heads * G, d)
    o, lse = attend(ec, q, c, n)
    check(o, lse, q, c, range(len(n)), n, d ** -0.5)


@pytest.mark.parametrize('e4m3', [False, True])
@pytest.mark.parametrize('splits', [0, 1, 2, 3, 7, 64, 1024])
def test_every_share_count(ec, splits, e4m3):
    n = [5000, 1, 700, 0, 4097, 64, 65]
    c = Cache(splits, n, 2, 128, 16, e4m3)
    q = query(splits, len(n), 8, 128)
    o, lse = attend(ec, q, c, n, shares=splits)
    check(o, lse, q, c, range(len(n)), n, 128 ** -0.5)


@pytest.mark.parametrize('window', [1, 15, 32, 100, 4096])
@pytest.mark.parametrize('splits', [None, 0, 9])
def test_windows(ec, window, splits):
    n = [3000, 1, 0, 32, 33, 99, 777]
    c = Cache(window, n, 4, 128, 16)
    for r, rows in enumerate(c.rows):       # what lies before the window is not to be read
        at = torch.arange(max(0, n[r] - window), device='cuda')
        c.cache[c.table[r].long()[at // 16], :, at % 16] = math.nan
    q = query(window, len(n), 8, 128)
    o, lse = attend(ec, q, c, n, window=window, shares=splits)
    check(o, lse, q, c, range(len(n)), n, 128 ** -0.5, window)


def test_many_tokens_share_requests(ec):
    """Chunks: every token of a request has its own length, the table is per request; requests out of order, odd numbers clamped."""
    n, chunk = [700, 40, 1300], [37, 1, 90]
    c = Cache(7, n, 2, 128, 32)
    requests = sum(([r] * k for r, k in zip((2, 0, 1), (90, 37, 1))), [])
    ctx = sum(([n[r] - k + i + 1 for i in range(k)] for r, k in zip((2, 0, 1), (90, 37, 1))), [])
    q = query(8, len(ctx), 8, 128)
    o, lse = ec.attention(q, c.cache, c.table, dev_i32(np.array(ctx)), 0.1, max(n), token_requests=dev_i64(np.array(requests)))
    check(o, lse, q, c, requests, ctx, 0.1)
    o, _ = ec.attention(q[:2], c.cache, c.table, dev_i32(np.array([30, 30])), 0.1, 30, token_requests=dev_i64(np.array([-5, 99])))
    check(o, ec.attention(q[:2], c.cache, c.table, dev_i32(np.array([30, 30])), 0.1, 30, token_requests=dev_i64(np.array([0, 2])))[1],
          q[:2], c, [0, 2], [30, 30], 0.1)


def test_strides(ec):
    """q out of a fused projection, a table with more columns, a cache inside a larger one."""
    n = [300, 17, 129]
    c = Cache(9, n, 4, 128, 16)
    wide = query(10, 3, 24, 128)
    big = torch.full((c.cache.shape[0], 16, 4, 3 * 256), math.nan, dtype=torch.bfloat16, device='cuda')
    big[..., 256:512] = c.cache.transpose(1, 2)
    table = torch.full((3, c.table.shape[1] + 5), 1 << 30, dtype=torch.int32, device='cuda')
    table[:, :c.table.shape[1]] = c.table
    q = wide[:, 4:12]
    o, lse = ec.attention(q, big[..., 256:512].transpose(1, 2), table[:, :c.table.shape[1]], dev_i32(np.array(n)), 0.09, 300)
    check(o, lse, q, c, range(3), n, 0.09)
    q = wide.transpose(0, 1)[:8].contiguous().transpose(0, 1)       # heads outermost
    o, lse = attend(ec, q, c, n)
    check(o, lse, q, c, range(3), n, 128 ** -0.5)


def test_lengths_past_the_table_and_pages_past_the_cache(ec):
    """A length counts up to the rows that the table holds; a negative one is none; page ids are clamped into the cache."""
    c = Cache(11, [64, 64, 64], 2, 64, 16, extra_cols=0)
    q = query(12, 3, 2, 64)
    o, lse = ec.attention(q, c.cache, c.table, dev_i32(np.array([1000, -3, 64])), 0.1, 1000)
    check(o, lse, q, c, range(3), [64, -3, 64], 0.1)
    c.cache[0] = c.cache[-1] = 0
    wild = c.table.clone()
    wild[0, 1], wild[2, 0] = -7, 1 << 30
    c.rows[0][16:32], c.rows[2][:16] = 0, 0
    o, lse = ec.attention(q, c.cache, wild, dev_i32(np.array([64, 64, 64])), 0.1, 64)
    check(o, lse, q, c, range(3), [64] * 3, 0.1)


def test_scales_of_scores(ec):
    """Sharp scores (one row takes all), scores that grow along the rows (the maximum is raised often), and a negative scale."""
    n = [2000, 500]
    c = Cache(13, n, 1, 128, 16)
    q = query(14, 2, 4, 128, 12.0)
    for scale in (0.5, -0.3, 1e-4, 0.0):
        o, lse = attend(ec, q, c, n, scale)
        if scale < 0:
            check(o, lse, -q, c, range(2), n, -scale)
        else:
            check(o, lse, q, c, range(2), n, scale)
    for r, rows in enumerate(c.rows):
        at = torch.arange(rows.shape[0], device='cuda')
        rows *= torch.linspace(0.01, 2, rows.shape[0], device='cuda').double()[:, None, None]
        rows.copy_(rows.to(torch.bfloat16).double())
        c.cache[c.table[r].long()[at // 16], :, at % 16] = rows.to(torch.bfloat16)
    o, lse = attend(ec, q, c, n, 0.5)
    check(o, lse, q, c, range(2), n, 0.5)


@pytest.mark.parametrize('splits', [0, 8])
def test_values_that_are_not_finite(ec, splits):
    """NaN in a row of K reaches output and lse of the heads that see it, NaN and infinities in V the output alone; -inf scores
    have no weight; a row of nothing else is an empty one. No other token, head or window sees any of it."""
    n = [600, 600, 600, 600, 40]
    c = Cache(15, n, 2, 128, 16)
    page = lambda r, j: (int(c.table[r, j // 16]), slice(None), j % 16)
    base = query(16, 5, 4, 128)
    base[3, :, 0], base[4, :, 0] = 1, 1
    p, _, x = page(0, 300)
    c.cache[p, 1, x, 5] = math.nan                       # K of KV head 1
    p, _, x = page(1, 599)
    c.cache[p, 0, x, 128 + 9] = math.inf                 # V of KV head 0
    p, _, x = page(2, 10)
    c.cache[p, 1, x, 128:] = math.nan
    p, _, x = page(3, 77)
    c.cache[p, :, x, 0] = -math.inf
    for j in range(40):
        p, _, x = page(4, j)
        c.cache[p, :, x, 0] = -math.inf
        c.cache[p, 1, x, 128:] = (math.nan, math.inf)[j % 2]      # values without any weight
    o, lse = attend(ec, base, c, n, shares=splits)
    assert torch.isnan(o[0, 2:]).all() and torch.isnan(lse[2:, 0]).all()
    assert torch.isposinf(o[1, :2, 9]).all() and torch.isnan(o[2, 2:]).all()
    assert torch.isfinite(o[1, :, :9]).all() and torch.isfinite(o[1, 2:]).all() and torch.isfinite(lse[:, 1:4]).all()
    assert (o[4] == 0).all() and torch.isneginf(lse[:, 4]).all()
    c.rows[3] = torch.cat((c.rows[3][:77], c.rows[3][78:]))
    for keep, t in ((slice(0, 2), 0), (slice(2, 4), 1), (slice(0, 2), 2), (slice(0, 4), 3)):
        part = Cache.__new__(Cache)
        part.h, part.rows = 1 if keep.stop - keep.start == 2 else 2, [c.rows[t][:, keep.start // 2:-(-keep.stop // 2)]]
        check(o[t:t + 1, keep].contiguous(), lse[keep, t:t + 1], base[t:t + 1, keep], part, [0], [c.rows[t].shape[0]], 128 ** -0.5)
    o, lse = attend(ec, base, c, n[:3] + [500] + [0], window=30, shares=splits)
    assert torch.isfinite(o[0]).all() and torch.isfinite(o[2:4]).all()      # the rows in question lie before the window


def test_same_bits_again(ec):
    n = [3000, 100, 2500]
    c = Cache(17, n, 4, 128, 16, True)
    q = query(18, 3, 8, 128)
    first = attend(ec, q, c, n)
    for _ in range(3):
        again = attend(ec, q, c, n)
        assert torch.equal(first[0], again[0]) and torch.equal(first[1], again[1])


def test_offsets_past_32_bits(ec):
    """Pages beyond 2^32 bytes, and a table whose rows lie far apart."""
    pages, h, d = 70000, 16, 128
    cache = torch.empty(pages, 16, h, 2 * d, dtype=torch.bfloat16, device='cuda')
    cache[-4:] = query(19, 4 * 16, h, 2 * d).view(4, 16, h, 2 * d)
    c = Cache.__new__(Cache)
    c.h, c.rows = h, [cache[[pages - 1, pages - 3]].flatten(0, 1).double()]
    table = dev_i32(np.array([[pages - 1, pages - 3]]))
    q = query(20, 1, h, d)
    o, lse = ec.attention(q, cache.transpose(1, 2), table, dev_i32(np.array([30])), 0.1, 32)
    check(o, lse, q, c, [0], [30], 0.1)
    key, value = query(21, 2, h, d), query(22, 2, h, d)
    ec.store_rows(key, value, dev_i64(np.array([pages * 16 - 1, pages * 16 - 17])), cache.transpose(1, 2))
    assert torch.equal(cache[-1, 15], torch.cat((key[0], value[0]), -1)) and torch.equal(cache[-2, 15], torch.cat((key[1], value[1]), -1))


def test_replayed_graphs(ec):
    """A captured step, replayed with other lengths, pages and queries; eager calls in between."""
    n = [900, 40, 2000, 0]
    c = Cache(23, n, 4, 128, 16)
    q, ctx = query(24, 4, 8, 128), dev_i32(np.array(n))
    call = lambda: ec.attention(q, c.cache, c.table, ctx, 0.1, 2000)
    call()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        o, lse = call()
    for seed, lengths in ((25, [3, 40, 1999, 0]), (26, [900, 0, 64, 0]), (27, [899, 39, 2000, 0])):
        q.copy_(query(seed, 4, 8, 128))
        ctx.copy_(dev_i32(np.array(lengths)))
        graph.replay()
        check(o, lse, q, c, range(4), lengths, 0.1)
        eager = call()
        torch.cuda.synchronize()
        assert torch.equal(eager[0], o) and torch.equal(eager[1], lse)


def test_streams_and_workspaces(ec, pkg):
    n = [4000, 3000]
    c = Cache(28, n, 2, 128, 16)
    q = query(29, 2, 4, 128)
    want = attend(ec, q, c, n, shares=16)
    ws = pkg.s6_ops.S6Workspace(4, 128, 2 * 16 + 1)
    got = attend(ec, q, c, n, shares=16, workspace=ws)
    assert torch.equal(want[0], got[0]) and torch.equal(want[1], got[1])
    with pytest.raises(RuntimeError, match='workspace overflow'):
        attend(ec, q, c, n, shares=17, workspace=ws)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = attend(ec, q, c, n, shares=16)
    side.synchronize()
    assert torch.equal(want[0], got[0])


def test_no_tokens(ec):
    c = Cache(30, [5], 2, 64, 16)
    o, lse = ec.attention(query(1, 0, 4, 64), c.cache, c.table[:0], dev_i32(np.zeros(0)), 0.1, 5)
    assert o.shape == (0, 4, 64) and lse.shape == (4, 0)
    ec.store_rows(query(1, 0, 2, 64), query(1, 0, 2, 64), dev_i64(np.zeros(0)), c.cache)
    o, lse = ec.attention(query(1, 2, 4, 64), c.cache, c.table.new_zeros(2, 0), dev_i32(np.array([5, 0])), 0.1, 5)
    assert (o == 0).all() and torch.isneginf(lse).all()


def test_refusals(ec):
    c = Cache(31, [5, 5], 2, 64, 16)
    q, n, t = query(1, 2, 4, 64), dev_i32(np.array([5, 5])), c.table
    scale = torch.ones(2, device='cuda')
    e4 = c.cache.to(E4)
    for args, match in (((q.float(), c.cache, t, n, 1.0, 5), 'bfloat16'), ((q, c.cache.float(), t, n, 1.0, 5), 'float8_e4m3fn'),
                        ((q[:, :3], c.cache, t, n, 1.0, 5), 'multiple of 2 heads'), ((q[0], c.cache, t, n, 1.0, 5), 'q must be'),
                        ((query(1, 2, 4, 128), c.cache, t, n, 1.0, 5), '64'), ((q, c.cache[0], t, n, 1.0, 5), 'exact cache'),
                        ((q, c.cache[..., :96], t, n, 1.0, 5), 'exact cache'), ((q, c.cache[:, :0], t, n, 1.0, 5), 'one KV head'), ((q, c.cache, t, n[:1], 1.0, 5), 'ctx'),
                        ((q, c.cache, t, n.long(), 1.0, 5), 'ctx'), ((q, c.cache, t[:1], n, 1.0, 5), 'block_table'),
                        ((q, c.cache, t.long(), n, 1.0, 5), 'block_table'), ((q, c.cache, t, n, 1.0, 5, n), 'token_requests'),
                        ((q, c.cache, t, n, 1.0, 5, None, -1), 'window'), ((q, c.cache, t, n, 1.0, 5, None, 0, scale), 'k_scale'),
                        ((q, e4, t, n, 1.0, 5, None, 0, None, scale[:1]), 'v_scale'), ((q, e4, t, n, 1.0, 5, None, 0, scale.half()), 'k_scale'),
                        ((q, c.cache, t, n, 1.0, 5, None, 0, None, None, 1025), 'shares'), ((q, c.cache, t, n, 1.0, 5, None, 0, None, None, -1), 'shares')):
        with pytest.raises(ValueError, match=match):
            ec.attention(*args)
    with pytest.raises(RuntimeError):
        ec.attention(q, c.cache, t.cpu(), n, 1.0, 5)
    rows, slots = query(2, 2, 2, 64), dev_i64(np.array([1, 2]))
    for args, match in (((rows, rows[:1], slots, c.cache), 'alike'), ((rows[:, :1], rows[:, :1], slots, c.cache), 'alike'),
                        ((rows, rows, slots[:1], c.cache), 'slots'), ((rows, rows, slots.int(), c.cache), 'slots'),
                        ((rows.half(), rows, slots, c.cache), 'bfloat16'), ((rows, rows, slots, c.cache, scale), 'k_scale')):
        with pytest.raises(ValueError, match=match):
            ec.store_rows(*args)


# ---- store -------------------------------------------------------------------------------------------------------------

def e4m3_of(x):
    """The nearest e4m3 value in 64 bits, ties to even, clamped to 448."""
    x = np.clip(x, -448, 448)
    step = 2.0 ** (np.floor(np.log2(np.maximum(np.abs(x), 2.0 ** -6))) - 3)
    return np.round(x / step) * step


@pytest.mark.parametrize('e4m3', [False, True])
@pytest.mark.parametrize('kv_heads,d,block,heads_first', [(16, 128, 16, False), (3, 64, 7, True), (1, 256, 1, False)])
def test_store(ec, kv_heads, d, block, heads_first, e4m3):
    """Every value of the cache, edges of the rounding among them, and nothing outside the slots; the divisions of fp32 can move a
    value to the neighbour only where it lies within 2^-24 of a tie, which the powers of two here do not."""
    T, pages = 40, 60 // block + 1
    wide = query(kv_heads + d, T, 2 * kv_heads + 1, d, 3.0)
    key, value = wide[:, 1:kv_heads + 1], wide[:, kv_heads + 1:]
    edges = torch.tensor([0., -0., 448, 449, 464, 465, -1e4, math.inf, -math.inf, math.nan, 2 ** -6, 2 ** -9, 2 ** -10, 3 * 2 ** -10, 17,
                          17.0625, 18, 19, 21, 1.0625, 1.1875, 240, 248, 432, 440, -17, -19, 2 ** -11, 2 ** -7, 0.0625, 1, -1], device='cuda')
    key[5, 0, :32], value[6, -1, :32] = edges.to(torch.bfloat16), edges.to(torch.bfloat16)
    slots = np.random.default_rng(d).permutation(pages * block)[:T].astype(np.int64)
    slots[[3, 11]] = -1
    slots[17], slots[18] = pages * block, 1 << 40
    shape = (pages, kv_heads, block, 2 * d) if heads_first else (pages, block, kv_heads, 2 * d)
    start = query(7, 1, int(np.prod(shape)) // 64, 64).view(shape).to(E4 if e4m3 else torch.bfloat16)
    cache = start.clone() if heads_first else start.clone().transpose(1, 2)
    scales = {}
    if e4m3:
        scales = dict(k_scale=2.0 ** torch.arange(kv_heads, device='cuda').float().remainder(3), v_scale=None if kv_heads == 3 else
                      2.0 ** -torch.arange(kv_heads, device='cuda').float().remainder(2))
    ec.store_rows(key, value, dev_i64(slots), cache, **scales)
    want = (start if heads_first else start.transpose(1, 2)).float().cpu().numpy().copy()
    for t, s in enumerate(slots):
        if 0 <= s < pages * block:
            for at, x, name in ((0, key, 'k_scale'), (d, value, 'v_scale')):
                x = x[t].double().cpu().numpy()
                if e4m3:
                    with np.errstate(invalid='ignore'):
                        x = e4m3_of(x / (1 if scales[name] is None else scales[name].cpu().numpy()[:, None]))
                want[s // block, :, s % block, at:at + d] = x
    assert np.array_equal(cache.float().cpu().numpy(), want, equal_nan=True)


def test_store_divides_by_the_scale(ec):
    """Scales that are no powers of two: within half a step of the quotient."""
    key, value = query(33, 500, 2, 64, 5.0), query(34, 500, 2, 64, 5.0)
    cache = torch.zeros(32, 2, 16, 128, device='cuda').to(E4)
    scale = torch.tensor([0.0173, 0.61], device='cuda')
    ec.store_rows(key, value, torch.arange(500, device='cuda'), cache, scale, scale)
    got = cache.float().transpose(1, 2).reshape(512, 2, 128)[:500].double()
    want = (torch.cat((key, value), -1).double() / scale.double()[:, None]).clamp(-448, 448)
    step = 2.0 ** (torch.floor(torch.log2(want.abs().clamp(min=2.0 ** -6))) - 3)
    assert ((got - want).abs() <= step / 2 * (1 + 2.0 ** -19)).all()


@pytest.mark.parametrize('e4m3', [False, True])
@pytest.mark.parametrize('T,kv_heads,G,d', [(300, 2, 1, 128), (150, 4, 12, 64), (70, 4, 3, 256), (500, 1, 16, 128), (1, 1, 128, 128),
                                           (1, 64, 1, 64), (2, 5, 20, 256)])
def test_many_tokens_and_many_heads(ec, T, kv_heads, G, d, e4m3):
    """Short rows of more groups than CUs, one token of many heads; all in one launch, and in shares."""
    n = np.random.default_rng(T).integers(0, 200, T).tolist()
    n[0] = 199
    c = Cache(T + G, n, kv_heads, d, 16, e4m3)
    q = query(T, T, kv_heads * G, d)
    for shares in (None, 5):
        o, lse = attend(ec, q, c, n, shares=shares)
        check(o, lse, q, c, range(T), n, d ** -0.5)


def test_a_token_of_a_very_long_row(ec):
    """More rows than shares of a workgroup's steps fit 16 bits; two KV heads."""
    n = [1200000, 3]
    c = Cache(60, n, 2, 64, 64, True)
    q = query(61, 2, 4, 64)
    o, lse = attend(ec, q, c, n)
    # (chains of up to 2^12 additions per lane and part: 2^-18 of the sums instead of the 2^-20 of the shorter rows)
    rows = c.rows[0]
    k, v = rows[..., :64].repeat_interleave(2, 1), rows[..., 64:].repeat_interleave(2, 1)
    s = (q[0].double() * k).sum(-1) / 8
    want_lse = torch.logsumexp(s, 0)
    p = torch.exp(s - want_lse)[..., None]
    want, size = (p * v).sum(0), (p * v.abs()).sum(0)
    e = 66 * 2.0 ** -24 / 8 * (q[0].double().abs() * k.abs()).sum(-1).amax(0)
    assert ((o[0].double() - want).abs() <= HALF * want.abs() + (2.0 ** -15 + 2.0 ** -18 + torch.expm1(2 * e))[:, None] * size).all()
    assert ((lse[:, 0].double() - want_lse).abs() <= e + 2.0 ** -18 + 2.0 ** -22 * want_lse.abs()).all()
    check(o[1:], lse[:, 1:], q[1:], c, [1], [3], 0.125)


# ---- tokens that go through the rows of a request together --------------------------------------------------------------

def chunks(n, lens, order):
    """Requests and lengths of the tokens of causal chunks, request after request."""
    requests = sum(([r] * lens[r] for r in order), [])
    return requests, sum(([n[r] - lens[r] + i + 1 for i in range(lens[r])] for r in order), [])


@pytest.mark.parametrize('e4m3', [False, True])
@pytest.mark.parametrize('kv_heads,G,d,block', [(2, 1, 128, 16), (1, 2, 64, 24), (2, 3, 128, 32), (1, 4, 256, 16), (1, 5, 64, 16),
                                               (2, 8, 128, 1), (3, 7, 128, 16)])
@pytest.mark.parametrize('window,turns', [(0, 1), (0, 4), (21, 2), (0, 16)])
def test_groups_of_tokens(ec, monkeypatch, kv_heads, G, d, block, e4m3, window, turns):
    """Chunks that begin and end inside a group of tokens, single tokens among them, tokens without rows, lengths in any order."""
    monkeypatch.setattr(ec, '_turns', lambda *a: turns)
    n, lens = [300, 40, 17, 900, 33], [37, 40, 1, 5, 33]
    c = Cache(G + d, n, kv_heads, d, block, e4m3)
    requests, ctx = chunks(n, lens, (3, 0, 1, 2, 4))
    ctx[7], ctx[60], ctx[-1] = 0, -4, 12
    requests, ctx = requests + [2, 0, 2], ctx + [17, 300, 5]
    assert len(ctx) >= 4 * len(n)
    q = query(G, len(ctx), kv_heads * G, d)
    o, lse = ec.attention(q, c.cache, c.table, dev_i32(np.array(ctx)), d ** -0.5, max(n), dev_i64(np.array(requests)), window,
                          c.k_scale, c.v_scale)
    check(o, lse, q, c, requests, ctx, d ** -0.5, window)


@pytest.mark.parametrize('e4m3', [False, True])
def test_rows_that_a_token_of_a_group_does_not_see(ec, monkeypatch, e4m3):
    """NaN and infinities in the rows behind a token's last, and before its window, reach only the tokens that see them."""
    monkeypatch.setattr(ec, '_turns', lambda *a: 3)
    n = [200]
    c = Cache(40, n, 2, 128, 16, e4m3)      # (one table row, sixteen tokens)
    ctx = [170, 171, 200, 172, 190, 1, 173, 174, 176, 177, 180, 179, 178, 175, 0, 169]
    requests = [0] * 15 + [0]
    base = query(41, 16, 4, 128)
    want = ec.attention(base, c.cache, c.table, dev_i32(np.array(ctx)), 0.1, 200, dev_i64(np.array(requests)), 0, c.k_scale, c.v_scale)
    check(*want, base, c, requests, ctx, 0.1)
    raw = c.cache.view(torch.uint8) if e4m3 else c.cache
    bad = 0x7F if e4m3 else math.nan
    at = torch.arange(176, 200, device='cuda')
    raw[c.table[0].long()[at // 16], :, at % 16] = bad
    o, lse = ec.attention(base, c.cache, c.table, dev_i32(np.array(ctx)), 0.1, 200, dev_i64(np.array(requests)), 0, c.k_scale, c.v_scale)
    sees = torch.tensor([x > 176 for x in ctx], device='cuda')
    assert torch.isnan(o[sees]).all() and torch.isnan(lse[:, sees]).all()
    assert torch.equal(o[~sees], want[0][~sees]) and torch.equal(lse[:, ~sees], want[1][:, ~sees])
    if not e4m3:
        c.cache[c.table[0, 176 // 16].long(), :, 176 % 16, 128:] = math.inf      # and an infinity in V alone
        c.cache[c.table[0, 176 // 16].long(), :, 176 % 16, :128] = 1
        o, lse = ec.attention(base, c.cache, c.table, dev_i32(np.array(ctx)), 0.1, 200, dev_i64(np.array(requests)), 0)
        assert torch.isposinf(o[ctx.index(177)]).all() and torch.isfinite(lse[:, ctx.index(177)]).all()
        assert torch.equal(o[~sees], want[0][~sees])
    raw[c.table[0].long()[at // 16], :, at % 16] = 0
    before = torch.arange(0, 150, device='cuda')
    window = 20
    clean = ec.attention(base, c.cache, c.table, dev_i32(np.array(ctx)), 0.1, 200, dev_i64(np.array(requests)), window, c.k_scale, c.v_scale)
    raw[c.table[0].long()[before // 16], :, before % 16] = bad
    o, lse = ec.attention(base, c.cache, c.table, dev_i32(np.array(ctx)), 0.1, 200, dev_i64(np.array(requests)), window, c.k_scale, c.v_scale)
    sees = torch.tensor([0 < x < 170 for x in ctx], device='cuda')
    assert torch.isnan(o[sees]).all() and torch.equal(o[~sees], clean[0][~sees]) and torch.equal(lse[:, ~sees], clean[1][:, ~sees])


def test_a_chunk_beside_single_tokens(ec):
    """Many single tokens and one chunk, through a table with rows to spare; the chunk's length as the hint."""
    n, lens = [400 + 13 * r for r in range(60)] + [900], [1] * 60 + [200]
    c = Cache(70, n, 16, 128, 16)
    requests, ctx = chunks(n, lens, range(61))
    q = query(71, len(ctx), 16, 128)
    table = torch.zeros(300, c.table.shape[1], dtype=torch.int32, device='cuda')
    table[:61] = c.table
    o, lse = ec.attention(q, c.cache, table, dev_i32(np.array(ctx)), 0.09, max(n), dev_i64(np.array(requests)), max_query_len=200)
    some = list(range(60)) + list(range(60, 260, 17)) + [259]
    check(o[some], lse[:, some], q[some], c, [requests[t] for t in some], [ctx[t] for t in some], 0.09)


@pytest.mark.parametrize('kv_heads,G', [(16, 1), (8, 4)])
def test_large_chunks(ec, kv_heads, G):
    """Steps large enough for groups by the rule, prompts without history among them."""
    n, lens = [1500, 700, 513, 3000], [300, 700, 1, 400]
    c = Cache(50 + G, n, kv_heads, 128, 16)
    requests, ctx = chunks(n, lens, range(4))
    assert ec._turns(len(ctx), G, kv_heads, 256, len(ctx) // 4) == 4
    q = query(51, len(ctx), kv_heads * G, 128)
    o, lse = ec.attention(q, c.cache, c.table, dev_i32(np.array(ctx)), 0.09, 3000, dev_i64(np.array(requests)))
    some = list(range(0, len(ctx), 61)) + [len(ctx) - 1]
    check(o[some], lse[:, some], q[some], c, [requests[t] for t in some], [ctx[t] for t in some], 0.09)
    alone = ec.attention(q, c.cache, c.table, dev_i32(np.array(ctx)), 0.09, 3000, dev_i64(np.array(requests)), shares=0)
    assert (o.float() - alone[0].float()).abs().max() <= 2.0 ** -6 * alone[0].float().abs().max()


@pytest.mark.parametrize('e4m3', [False, True])
@pytest.mark.parametrize('kv_heads,G,d,block', [(128, 1, 128, 16), (64, 2, 64, 24), (43, 3, 128, 32), (26, 5, 64, 16), (18, 8, 128, 1),
                                                (18, 7, 128, 16), (18, 8, 256, 16)])
@pytest.mark.parametrize('window,turns', [(0, 1), (0, 4), (21, 16)])
def test_groups_where_there_are_many(ec, monkeypatch, kv_heads, G, d, block, e4m3, window, turns):
    """As above with two workgroups per CU (for groups of twice the tokens): chunks that end inside a group, single tokens, none."""
    monkeypatch.setattr(ec, '_turns', lambda *a: turns)
    n, lens = [300, 40, 17, 900, 33], [37, 40, 1, 5, 33]
    c = Cache(G + d, n, kv_heads, d, block, e4m3)
    requests, ctx = chunks(n, lens, (3, 0, 1, 2, 4))
    ctx[7], ctx[60], ctx[-1] = 0, -4, 12
    requests, ctx = requests + [2, 0, 2], ctx + [17, 300, 5]
    assert -(-len(ctx) // (32 // G)) * kv_heads >= 512
    q = query(G, len(ctx), kv_heads * G, d)
    o, lse = ec.attention(q, c.cache, c.table, dev_i32(np.array(ctx)), d ** -0.5, max(n), dev_i64(np.array(requests)), window,
                          c.k_scale, c.v_scale)
    check(o, lse, q, c, requests, ctx, d ** -0.5, window)


@pytest.mark.parametrize('e4m3', [False, True])
def test_rows_that_a_token_of_many_does_not_see(ec, monkeypatch, e4m3):
    """NaN behind a token's last row and before its window reach only the tokens that see them, in groups of 32 tokens."""
    monkeypatch.setattr(ec, '_turns', lambda *a: 1)
    n = [200]
    c = Cache(42, n, 512, 64, 16, e4m3)
    ctx = [170 + 7 * i % 31 for i in range(30)] + [0, 1]
    table_rows, lengths = dev_i64(np.zeros(32)), dev_i32(np.array(ctx))
    q = query(43, 32, 512, 64)
    run = lambda window: ec.attention(q, c.cache, c.table, lengths, 0.1, 200, table_rows, window, c.k_scale, c.v_scale)
    raw = c.cache.view(torch.uint8) if e4m3 else c.cache
    bad = 0x7F if e4m3 else math.nan
    clean = run(0), run(20)
    check(*clean[0], q, c, [0] * 32, ctx, 0.1)
    check(*clean[1], q, c, [0] * 32, ctx, 0.1, 20)
    saved = raw.clone()
    for at, window, sees in ((range(176, 200), 0, [x > 176 for x in ctx]), (range(160), 20, [0 < x < 180 for x in ctx])):
        at = torch.tensor(at, device='cuda')
        raw[c.table[0].long()[at // 16], :, at % 16] = bad
        o, lse = run(window)
        sees = torch.tensor(sees, device='cuda')
        assert torch.isnan(o[sees]).all() and torch.isnan(lse[:, sees]).all()
        seen_by_none = [i for i in range(32) if not sees[i]]
        check(o[seen_by_none], lse[:, seen_by_none], q[seen_by_none], c, [0] * 32, [ctx[i] for i in seen_by_none], 0.1, window)
        raw.copy_(saved)
