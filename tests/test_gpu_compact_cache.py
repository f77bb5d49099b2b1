"""The compact latent cache and eviction on the GPU against the plain 64-bit restatement (``compact_ref``).

Tolerances. The kernel's weights and its output are each rounded to bf16 (half a step: 2^-8 relative), so an output is off
by at most 2^-8 (sum p |v| + |o|); its fp32 scores are off by at most (w + 2) 2^-24 scale sum |q k| =: d, which moves a
weight by a factor of up to exp(2 d); exponentials and sums add 2^-20 of the sum at the sizes here (up to 2^11 terms in
chains of at most 2^4 additions per lane, 2^-24 each, and 2^-22 per exponential). The log-sum-exp is off by d, those sums and its own rounding."""
import math

import numpy as np
import pytest
import torch

import compact_ref as C
from s6util import FakeLatentLayer, dev_bf16, dev_i32, dev_i64, host_f32, random_bits
from oracle import bf16

pytestmark = pytest.mark.gpu
SCALE = 1 / math.sqrt(128)
HALF = 2.0 ** -8


@pytest.fixture(scope='module')
def cc(pkg):
    return pkg.compact_cache


def dev_u8(a):
    return torch.from_numpy(np.ascontiguousarray(a)).cuda()


def host_u8(t):
    return t.cpu().numpy()


def latents(rng, shape):
    """Rows whose columns differ in size, as bf16 bits."""
    size = np.exp(0.5 * rng.standard_normal(shape[-1]))
    return bf16.from_f32(np.asarray(rng.standard_normal(shape) * size, np.float32))


class Pool:
    """Requests of given lengths in a compact cache with random pages; everything outside their rows reads as NaN."""

    def __init__(self, rng, lengths, width, block, extra_cols=1, spare=2):
        self.n, self.w, self.block = np.asarray(lengths), width, block
        cols = -(-max(max(lengths), 1) // block) + extra_cols
        pages = len(lengths) * cols + spare
        self.table = rng.permutation(np.arange(spare, pages))[:len(lengths) * cols].reshape(-1, cols).astype(np.int32)
        self.cache = np.full((pages, block // 16, 17 * width), 255, np.uint8)
        for r, n in enumerate(lengths):
            rows = bf16.to_f32(latents(rng, (n, 2 * width)))
            C.store(self.cache, rows[:, :width], rows[:, width:], C.slots_of(self.table[r], block, n))

    def rows(self, r, n=None):
        return C.load(self.cache, C.slots_of(self.table[r], self.block, self.n[r] if n is None else n))


def check_attention(o, lse, q, rows_of, ctx):
    """o [T, 16, w], lse [16, T] against float64, with the bounds above."""
    w = q.shape[-1]
    for t, n in enumerate(ctx):
        rows = rows_of(t)[:n]
        want, want_lse, size = C.attention(q[t].astype(np.float64), rows, SCALE)
        d = (w + 2) * 2.0 ** -24 * SCALE * (np.abs(q[t]).astype(np.float64) @ np.abs(rows[:, :w]).T).max() if n else 0.0
        bound = HALF * (size * 1.01 + np.abs(want)) + (math.expm1(2 * d) + 2.0 ** -20) * size
        assert (np.abs(o[t] - want) <= bound).all(), (t, n, float((np.abs(o[t] - want) - bound).max()))
        if n == 0:
            assert np.isneginf(lse[:, t]).all() and (o[t] == 0).all()
        else:
            assert (np.abs(lse[:, t] - want_lse) <= d + 2.0 ** -20 + 2.0 ** -22 * np.abs(want_lse)).all(), (t, n)


# ---- rows in and out ---------------------------------------------------------------------------------------------

@pytest.mark.parametrize('width,block', [(128, 16), (256, 32), (512, 16), (512, 48), (1024, 16)])
def test_stored_bytes(cc, width, block):
    """Every byte of the cache, values at the borders of the rounding among them, and nothing outside the slots."""
    rng = np.random.default_rng(width + block)
    T, pages = 45, 5
    key, value = latents(rng, (T, width)), latents(rng, (T, width))
    edges = np.array([0, -0.0, 0.25, -0.25, 0.2500001, 0.75, 1.25, 1.75, 2.5, 3.5, 5, 6, 6.5, 7, -7, 7.03125, 8, 0.125, 4,
                      -5, 3, 1, 2, 0.5, -1.5, -0.75, -2.5, -3.5, 1e-3, -6, 5.03125, 4.96875], np.float32)
    for t, top in enumerate((7, 7.03125, 6, 8)):     # a block's largest value decides its scale
        key[t, :32] = bf16.from_f32(np.where(np.abs(edges) < top, edges, top).astype(np.float32))
    key[4, :32] = bf16.from_f32(edges * np.float32(2.0 ** -118))
    key[5, :32] = bf16.from_f32(edges * np.float32(2.0 ** -127))   # below the smallest scale
    key[6, :32] = bf16.from_f32(edges * np.float32(2.0 ** 124))
    key[7, :32] = 0x7F7F                                          # the largest bf16
    key[8, 3], value[9, 40], value[10, 96] = 0x7F80, 0xFF80, 0x7FC1
    value[11], key[12] = 0, 0x8000
    key[13, :32] = 1                                              # the smallest denormal
    slots = rng.permutation(pages * block)[:T].astype(np.int64)
    slots[20], slots[21], slots[22] = -1, pages * block, pages * block + 77
    start = rng.integers(0, 256, (pages, block // 16, 17 * width)).astype(np.uint8)
    want = start.copy()
    C.store(want, bf16.to_f32(key), bf16.to_f32(value), slots)
    cache = dev_u8(start)
    cc.store_rows(dev_bf16(key), dev_bf16(value), dev_i64(slots), cache)
    assert (host_u8(cache) == want).all()


def test_store_takes_strides_and_single_rows(cc):
    rng = np.random.default_rng(3)
    w, block = 256, 16
    bits = latents(rng, (9, 2 * w + 3))
    want = np.zeros((3, 1, 17 * w), np.uint8)
    slots = np.arange(9, dtype=np.int64) * 5
    C.store(want, bf16.to_f32(bits[:, 1:w + 1]), bf16.to_f32(bits[:, w + 2:2 * w + 2]), slots)
    wide = dev_bf16(bits)                                         # odd strides, rows that are not 16-byte aligned
    cache = torch.zeros(3, 1, 17 * w, dtype=torch.uint8, device='cuda')
    cc.store_rows(wide[:, 1:w + 1], wide[:, w + 2:2 * w + 2], dev_i64(slots), cache)
    assert (host_u8(cache) == want).all()
    pages = torch.zeros(6, 1, 17 * w, dtype=torch.uint8, device='cuda')
    for t in range(9):                                            # row by row, in every other page of a pool
        cc.store_rows(wide[t:t + 1, 1:w + 1], wide[t:t + 1, w + 2:2 * w + 2], dev_i64(slots[t:t + 1]), pages[::2])
    assert (host_u8(pages[::2]) == want).all() and not host_u8(pages[1::2]).any()
    cc.store_rows(wide[:0, :w], wide[:0, :w], dev_i64([]), cache)
    assert (host_u8(cache) == want).all()


@pytest.mark.parametrize('width,block', [(128, 16), (256, 48), (512, 16), (1024, 32)])
def test_loaded_rows(cc, width, block):
    rng = np.random.default_rng(width)
    lengths = [37, 0, 1, 64, 16]
    p = Pool(rng, lengths, width, block)
    out = host_f32(cc.load_rows(dev_u8(p.cache), dev_i32(p.table), dev_i32(lengths), 65))
    assert out.shape == (5, 65, 2 * width)
    for r, n in enumerate(lengths):
        assert (out[r, :n] == p.rows(r)).all() and (out[r, n:] == 0).all()
    wide = torch.full((5, 40, 2 * width + 8), 7., dtype=torch.bfloat16, device='cuda')
    cc.load_rows(dev_u8(p.cache), dev_i32(p.table), dev_i32(lengths), 39, out=wide[:, 1:, :2 * width])
    got = host_f32(wide)
    for r, n in enumerate(lengths):
        assert (got[r, 1:1 + min(n, 39), :2 * width] == p.rows(r, min(n, 39))).all()
        assert (got[r, 1 + min(n, 39):, :2 * width] == 0).all()
    assert (got[:, 0] == 7).all() and (got[:, :, 2 * width:] == 7).all()


def test_page_ids_outside_the_cache(cc):
    """Bad table entries are kept inside the cache, lengths past the table inside the table."""
    rng = np.random.default_rng(5)
    p = Pool(rng, [40], 128, 16, extra_cols=0)
    cache, table = dev_u8(p.cache), dev_i32([[-7, 10 ** 9, int(p.table[0, 2])]])
    out = host_f32(cc.load_rows(cache, table, dev_i32([10 ** 6]), 60))
    last = C.load(p.cache, np.arange(16) + 16 * (len(p.cache) - 1))
    assert np.array_equal(out[0, 16:32], last, equal_nan=True) and (out[0, 48:] == 0).all()
    assert np.array_equal(out[0, 32:40], p.rows(0)[32:40])
    q = dev_bf16(random_bits(rng, (1, 16, 128)))
    o, lse = cc.history_attention(q, cache, table, dev_i32([10 ** 6]), SCALE, 48)
    assert o.shape == (1, 16, 128) and lse.shape == (16, 1)
    o, lse = cc.history_attention(q, cache, table, dev_i32([-3]), SCALE, 48)
    assert (o == 0).all() and torch.isneginf(lse).all()


# ---- attention -----------------------------------------------------------------------------------------------------

@pytest.mark.parametrize('splits', [None, 1, 5])
@pytest.mark.parametrize('width,block', [(128, 16), (256, 16), (512, 48), (1024, 32)])
def test_history_attention(cc, width, block, splits):
    rng = np.random.default_rng(width + block)
    ctx = [700, 129, 17, 1, 0, 16, 33, 128, 250, 31, 511, 64]
    p = Pool(rng, ctx, width, block)
    q = random_bits(rng, (len(ctx), 16, width), 1.4 * math.sqrt(128 / width))
    o, lse = cc.history_attention(dev_bf16(q), dev_u8(p.cache), dev_i32(p.table), dev_i32(ctx), SCALE, 700,
                                  num_kv_splits=splits)
    check_attention(host_f32(o), host_f32(lse), bf16.to_f32(q), p.rows, ctx)


@pytest.mark.parametrize('splits', [2, 31, 64, 1024])
@pytest.mark.parametrize('width', [128, 256, 512, 1024])
def test_reduction_over_slots(cc, width, splits):
    """Few and many slots, most of them without rows; a row without any; a strided order of tokens in the table."""
    rng = np.random.default_rng(width + splits)
    ctx = [1700, 0, 33, 64]
    p = Pool(rng, ctx, width, 16)
    q = random_bits(rng, (4, 16, width), 1.4 * math.sqrt(128 / width))
    order = np.array([2, 0, 3, 1])
    o, lse = cc.history_attention(dev_bf16(q), dev_u8(p.cache), dev_i32(p.table), dev_i32(np.array(ctx)[order]), SCALE, 1700,
                                  token_requests=dev_i64(order), num_kv_splits=splits)
    check_attention(host_f32(o), host_f32(lse), bf16.to_f32(q), lambda t: p.rows(order[t]), np.array(ctx)[order])


@pytest.mark.parametrize('splits', [1, 4, 100])
def test_rows_that_read_as_nan(cc, splits):
    """A NaN among a request's rows makes its output and lse NaN, in one slot or in every one, and no other request's."""
    rng = np.random.default_rng(21)
    p = Pool(rng, [500, 500, 500], 256, 16)
    for r, rows in ((0, [499]), (1, np.arange(500))):
        bad = np.full((len(rows), 256), np.nan)
        C.store(p.cache, bad, bad, C.slots_of(p.table[r], 16, 500)[rows])
    q = random_bits(rng, (3, 16, 256))
    o, lse = cc.history_attention(dev_bf16(q), dev_u8(p.cache), dev_i32(p.table), dev_i32([500] * 3), SCALE, 500, num_kv_splits=splits)
    assert torch.isnan(o[:2]).all() and torch.isnan(lse[:, :2]).all()
    check_attention(host_f32(o)[2:], host_f32(lse)[:, 2:], bf16.to_f32(q)[2:], lambda t: p.rows(2), [500])


def test_history_of_one_request_and_of_many(cc):
    rng = np.random.default_rng(8)
    for ctx in ([1500], [5] * 70, [300] * 40 + [0] * 3):
        p = Pool(rng, ctx, 256, 16)
        q = random_bits(rng, (len(ctx), 16, 256))
        o, lse = cc.history_attention(dev_bf16(q), dev_u8(p.cache), dev_i32(p.table), dev_i32(ctx), SCALE, max(ctx))
        check_attention(host_f32(o), host_f32(lse), bf16.to_f32(q), p.rows, ctx)


def test_history_per_request_tables_plans_and_strides(cc, ops):
    """Tokens of requests through a per-request table, with a step's plan, a workspace, and a strided query."""
    rng = np.random.default_rng(9)
    p = Pool(rng, [333, 20, 150], 512, 16)
    req = np.array([0, 0, 0, 1, 2, 2])
    ctx = np.array([333, 333, 300, 20, 150, 0])
    wide = random_bits(rng, (6, 18, 520), 0.7)
    q = dev_bf16(wide)[:, 1:17, 8:]
    cache, table, c = dev_u8(p.cache), dev_i32(p.table), dev_i32(ctx)
    ws = ops.S6Workspace(16, 512, 6 * 6)
    want = None
    for splits, plan in ((6, None), (6, ops.split_plan(c, p.table.shape[1] * 16, 6)),
                         (6, ops.split_plan(c, p.table.shape[1] * 16, 6, dev_i32([0, 3, 4, 6])))):
        o, lse = cc.history_attention(q, cache, table, c, SCALE, 333, token_requests=dev_i64(req), num_kv_splits=splits,
                                      workspace=ws, plan=plan)
        check_attention(host_f32(o), host_f32(lse), bf16.to_f32(wide)[:, 1:17, 8:], lambda t: p.rows(req[t]), ctx)
        want = (o, lse) if want is None else want
        assert torch.equal(o, want[0]) and torch.equal(lse, want[1])   # a plan changes who does the work, not the sums
    parts = cc.history_partials(q, cache, table, c, SCALE, 6, ws, token_requests=dev_i64(req))
    o, lse = ops.history_reduce(parts)   # the bf16 cache's reduction: the same slots, another order
    check_attention(host_f32(o), host_f32(lse), bf16.to_f32(wide)[:, 1:17, 8:], lambda t: p.rows(req[t]), ctx)


@pytest.mark.parametrize('width', [128, 256, 512, 1024])
def test_prompt_chunks(cc, width):
    """Chunks share their rows through one expansion: ragged chunks, an empty request, padding tokens, NaN behind the rows."""
    rng = np.random.default_rng(width + 1)
    n, chunk = [210, 0, 33, 97], [20, 17, 1, 30]
    p = Pool(rng, n, width, 16)
    start = np.concatenate(([0], np.cumsum(chunk)))
    req = np.concatenate((np.repeat(np.arange(4), chunk), [3, 3]))     # two padding tokens, clamped to the last request
    ctx = np.concatenate((np.repeat(n, chunk), [0, 0]))
    q = random_bits(rng, (len(req), 16, width), math.sqrt(128 / width))
    o, lse = cc.history_attention(dev_bf16(q), dev_u8(p.cache), dev_i32(p.table), dev_i32(ctx), SCALE, 210,
                                  token_requests=dev_i64(req), query_start_loc=dev_i32(start), max_query_len=30)
    check_attention(host_f32(o), host_f32(lse), bf16.to_f32(q), lambda t: p.rows(req[t]), ctx)


@pytest.mark.parametrize('splits', [1, 3])
@pytest.mark.parametrize('width,block', [(256, 48), (512, 16), (1024, 32)])
def test_two_tokens_together(cc, monkeypatch, width, block, splits):
    """Pairs of one request, pairs that differ in request or length, an odd token at the end, rows of NaN in one request that
    the other token of its pair must not see, rows longer than the pages a wave looks up at a time."""
    monkeypatch.setattr(cc, 'history_shape', lambda *a: (2, splits))
    rng = np.random.default_rng(width + splits)
    n, chunk = [1100 if width == 256 else 530, 49, 20, 0, 64], [5, 3, 1, 2, 4]
    p = Pool(rng, n, width, block)
    C.store(p.cache, np.full((3, width), np.nan), np.full((3, width), np.nan), C.slots_of(p.table[1], block, 49)[[0, 17, 48]])
    req = np.repeat(np.arange(5), chunk)
    ctx = np.array(n)[req]
    ctx[[1, 13]] = 33, 0
    q = random_bits(rng, (len(req), 16, width), 1.4 * math.sqrt(128 / width))
    args = (dev_bf16(q), dev_u8(p.cache), dev_i32(p.table), dev_i32(ctx), SCALE)
    o, lse = cc.history_attention(*args, max(n), token_requests=dev_i64(req), max_query_len=5)
    bad = req == 1
    assert torch.isnan(o[torch.from_numpy(bad)]).all() and torch.isnan(lse[:, torch.from_numpy(bad)]).all()
    keep = np.flatnonzero(~bad)
    check_attention(host_f32(o)[keep], host_f32(lse)[:, keep], bf16.to_f32(q)[keep], lambda t: p.rows(req[keep[t]]), ctx[keep])
    again = cc.history_attention(*args, max(n), token_requests=dev_i64(req), max_query_len=5)
    assert torch.equal(o[keep], again[0][keep])


def test_rows_expanded_once(cc, monkeypatch):
    """The rows of chunks through one expansion to bf16: ragged chunks, an empty request, padding tokens, NaN behind the rows."""
    monkeypatch.setattr(cc, 'history_shape', lambda *a: (3, 1))
    rng = np.random.default_rng(11)
    n, chunk, width = [210, 0, 33, 97], [20, 17, 1, 30], 512
    p = Pool(rng, n, width, 16)
    start = np.concatenate(([0], np.cumsum(chunk)))
    req = np.concatenate((np.repeat(np.arange(4), chunk), [3, 3]))
    ctx = np.concatenate((np.repeat(n, chunk), [0, 0]))
    q = random_bits(rng, (len(req), 16, width), 0.5)
    o, lse = cc.history_attention(dev_bf16(q), dev_u8(p.cache), dev_i32(p.table), dev_i32(ctx), SCALE, 210,
                                  token_requests=dev_i64(req), query_start_loc=dev_i32(start), max_query_len=30)
    check_attention(host_f32(o), host_f32(lse), bf16.to_f32(q), lambda t: p.rows(req[t]), ctx)


@pytest.mark.parametrize('shape', [(1, 2), (2, 1), (2, 3), (3, 1)])
def test_captured_chunks(cc, monkeypatch, shape):
    """Every form of a chunk step in a graph: replays with new queries and lengths, eager work between them, equal the eager
    results bit for bit."""
    monkeypatch.setattr(cc, 'history_shape', lambda *a: shape)
    rng = np.random.default_rng(31)
    n, chunk = [130, 60], [7, 6]
    p = Pool(rng, n, 512, 16)
    req = np.repeat([0, 1], chunk)
    q, ctx = dev_bf16(random_bits(rng, (13, 16, 512), 0.5)), dev_i32(np.array(n)[req])
    cache, table, start, treq = dev_u8(p.cache), dev_i32(p.table), dev_i32([0, 7, 13]), dev_i64(req)
    call = lambda: cc.history_attention(q, cache, table, ctx, SCALE, 130, token_requests=treq, query_start_loc=start, max_query_len=7)
    call()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        o, lse = call()
    for turn in range(3):
        q.copy_(dev_bf16(random_bits(rng, (13, 16, 512), 0.5)))
        ctx.copy_(dev_i32(np.maximum(np.array(n)[req] - 9 * turn, 0)))
        o.fill_(float('nan'))
        graph.replay()
        want, want_lse = call()
        torch.cuda.synchronize()
        assert torch.equal(o, want) and torch.equal(lse, want_lse)
    check_attention(host_f32(o), host_f32(lse), host_f32(q), lambda t: p.rows(req[t]), ctx.cpu().numpy())


@pytest.mark.parametrize('width,n', [(256, 60), (512, 4200), (1024, 40)])
def test_steps_of_many_tokens(cc, width, n):
    """Steps that take two tokens a workgroup by their own size (and, with long rows, few tokens), beside the kernel for one."""
    rng = np.random.default_rng(width)
    T = 600 if n < 4096 else 40
    p = Pool(rng, [n, n // 2], width, 16)
    req = np.arange(T) // (T // 2 + 1)
    ctx = np.array([n, n // 2])[req]
    q = dev_bf16(random_bits(rng, (T, 16, width), 1.4 * math.sqrt(128 / width)))
    assert cc.history_shape(n, T, 2, 256, width)[0] == 2
    call = lambda length: cc.history_attention(q, dev_u8(p.cache), dev_i32(p.table), dev_i32(ctx), SCALE, n,
                                               token_requests=dev_i64(req), max_query_len=length)
    o, lse = call(T // 2 + 1)
    o1, lse1 = call(1)
    some = [0, 1, T // 2, T // 2 + 1, T - 1]
    rows = {t: p.rows(req[t]) for t in some}
    for a, b in ((o, lse), (o1, lse1)):
        check_attention(host_f32(a[some]), host_f32(b[:, some]), host_f32(q[some]), lambda i: rows[some[i]], ctx[some])
    assert (o.float() - o1.float()).norm() <= 2 * HALF * o.float().norm()   # each output of the two is off by 2^-8 twice
    assert (lse - lse1).abs().max() <= 1e-4


def test_rows_past_four_gigabytes(cc):
    """Offsets that pass 32 bits: the rows lie in the last pages of a pool of over 4 GiB."""
    rng = np.random.default_rng(10)
    w, pages = 1024, 250_000
    cache = torch.empty(pages, 1, 17 * w, dtype=torch.uint8, device='cuda')
    assert (pages - 4) * 17 * w > 2 ** 32
    rows, table = latents(rng, (50, 2 * w)), np.arange(pages - 4, pages, dtype=np.int32)[None]
    bits = dev_bf16(rows)
    cc.store_rows(bits[:, :w], bits[:, w:], dev_i64(C.slots_of(table[0], 16, 50)), cache)
    small = np.zeros((4, 1, 17 * w), np.uint8)
    C.store(small, bf16.to_f32(rows[:, :w]), bf16.to_f32(rows[:, w:]), np.arange(50))
    want = C.load(small, np.arange(50))
    assert (host_f32(cc.load_rows(cache, dev_i32(table), dev_i32([50]), 50))[0] == want).all()
    q = random_bits(rng, (1, 16, w), 0.4)
    o, lse = cc.history_attention(dev_bf16(q), cache, dev_i32(table), dev_i32([50]), SCALE, 50)
    check_attention(host_f32(o), host_f32(lse), bf16.to_f32(q), lambda t: want, [50])
    cc.move_rows(cache, dev_i32(table), cc.Eviction(None, None, None, dev_i32([[49]]), dev_i32([[0]])))
    assert (host_f32(cc.load_rows(cache, dev_i32(table), dev_i32([1]), 1))[0, 0] == want[49]).all()


# ---- accounts ------------------------------------------------------------------------------------------------------

def want_account(start, q, rows, w, lse, req, ctx, limit):
    """Float64 account, and how far off a kernel may be: its scores by d, the difference to the lse and the exponential by
    2^-21 (1 + |log p|) at the magnitudes here, and a sum of 16 heads per token in chains of at most 2^10 by 2^-14."""
    out, bound = start.astype(np.float64), np.abs(start) * 2.0 ** -23
    for t, r in enumerate(req):
        n = min(ctx[t], limit)
        if n == 0:
            continue
        k = rows(r)[:n, :w]
        s = q[t].astype(np.float64) @ k.T * SCALE
        d = (w + 2) * 2.0 ** -24 * SCALE * (np.abs(q[t]).astype(np.float64) @ np.abs(k).T)
        p = np.where(np.isinf(lse[:, t])[:, None], 0, np.exp(s - np.where(np.isinf(lse[:, t]), 0, lse[:, t])[:, None]))
        out[r, :n] += p.sum(0)
        bound[r, :n] += (p * (d * 1.01 + 2.0 ** -21 * (1 + np.abs(s) + np.abs(np.where(p > 0, lse[:, t][:, None], 0)))
                              + 2.0 ** -14)).sum(0)
    return out, bound


@pytest.mark.parametrize('compact', [True, False])
@pytest.mark.parametrize('width,block,chunk', [(128, 16, 1), (512, 16, 1), (256, 32, 3), (512, 48, 37), (1024, 16, 1),
                                               (1024, 16, 40), (256, 16, 70)])
def test_attention_weights(cc, width, block, chunk, compact):
    rng = np.random.default_rng(width + chunk)
    n = [200, 1, 0, 77, 130]
    p = Pool(rng, n, width, block)
    rows = p.rows
    cache = dev_u8(p.cache)
    if not compact:   # the same rows as bf16 pages
        pages = len(p.cache)
        every = C.load(p.cache, np.arange(pages * block))
        cache = torch.from_numpy(every.reshape(pages, 1, block, 2 * width)).to(torch.bfloat16).cuda()
    req = np.concatenate((np.repeat(np.arange(5), chunk), [4]))         # and a padding token
    ctx = np.concatenate((np.repeat(n, chunk), [50]))
    ctx[1] = min(ctx[1], 150)
    T = len(req)
    q = random_bits(rng, (T, 16, width), 1.4 * math.sqrt(128 / width))
    lse = rng.standard_normal((16, T)).astype(np.float32) + 8
    lse[:, 0] += 4
    lse[3, 0], lse[4, 0] = -np.inf, np.inf
    M = 190
    start = rng.random((5, M + 2)).astype(np.float32)
    want, bound = want_account(start[:, :M], bf16.to_f32(q), rows, width, lse, req[:-1], ctx, M)
    qsl = dev_i32(np.arange(0, T, chunk))
    got = []
    for _ in range(2):
        account = torch.from_numpy(start).cuda()
        out = cc.attention_weights(dev_bf16(q), cache, dev_i32(p.table), qsl, dev_i32(ctx), torch.from_numpy(lse).cuda(),
                                   SCALE, account[:, :M])
        assert out.data_ptr() == account.data_ptr()
        got.append(account)
    assert torch.equal(got[0], got[1]), 'the same call gave other bits'
    got = got[0].cpu().numpy()
    assert (got[:, M:] == start[:, M:]).all()
    for r in range(5):
        assert (got[r, min(n[r], M):M] == start[r, min(n[r], M):M]).all()   # rows behind the request
    assert (np.abs(got[:, :M] - want) <= bound).all(), float((np.abs(got[:, :M] - want) - bound).max())


def test_attention_weights_sum_to_the_softmax(cc):
    """With the history's own lse every token gives its 16 heads' weight of 1 to its request's rows."""
    rng = np.random.default_rng(12)
    n = [900, 310]
    for chunk in (1, 64):
        p = Pool(rng, n, 256, 16)
        T = 2 * chunk
        req, ctx = np.repeat([0, 1], chunk), np.repeat(n, chunk)
        q, cache, table = dev_bf16(random_bits(rng, (T, 16, 256))), dev_u8(p.cache), dev_i32(p.table)
        _, lse = cc.history_attention(q, cache, table, dev_i32(ctx), SCALE, 900, token_requests=dev_i64(req))
        account = cc.attention_weights(q, cache, table, dev_i32([0, chunk, T]), dev_i32(ctx), lse, SCALE,
                                       torch.zeros(2, 900, device='cuda'))
        # one relative error of at most 2^-14 (as above) per weight
        assert (account.sum(1).cpu() - 16 * chunk).abs().max() <= 16 * chunk * 2.0 ** -13


# ---- selection and moves --------------------------------------------------------------------------------------------

def run_select(cc, weights, positions, lengths, budget, protect):
    dev = lambda a: torch.from_numpy(np.ascontiguousarray(a)).cuda()
    b = dev(budget.astype(np.int32)) if isinstance(budget, np.ndarray) else budget
    w, pos = dev(weights), dev(positions)
    e = cc.select_rows(w, pos, dev_i32(lengths), b, dev_i32(protect))
    assert torch.equal(w.view(torch.int32), dev(weights).view(torch.int32)) and torch.equal(pos, dev(positions))
    budgets = budget if isinstance(budget, np.ndarray) else np.full(len(lengths), budget)
    for got, want, name in zip(e, C.select(weights, positions, lengths, budgets, protect), e._fields):
        got = got.cpu().numpy()
        assert got.shape == want.shape and np.array_equal(got, want, equal_nan=got.dtype.kind == 'f'), name
    return e


@pytest.mark.parametrize('M', [1, 2, 100, 2047, 2500, 8192, 9000])
def test_select_rows(cc, M):
    rng = np.random.default_rng(M)
    R = 6
    weights = np.exp(3 * rng.standard_normal((R, M))).astype(np.float32)
    weights[1] = rng.integers(0, 3, M)                          # ties everywhere
    weights[2] = 1
    weights[3, ::3] = 0
    weights[4, rng.integers(0, M, 5)] = [np.nan, np.inf, -np.inf, -0.0, -2]
    weights[5] = -weights[5]
    positions = (3 * np.argsort(rng.random((R, M)) + np.arange(M) / 16, -1)).astype(np.int32)
    lengths = np.array([M, M, M - 1, max(M // 2, 1), M, M])
    protect = (3 * (lengths - min(20, M // 3))).astype(np.int64)
    run_select(cc, weights, positions, lengths, max(1, M // 2), protect)
    run_select(cc, weights, positions, lengths, np.array([0, M // 3, M, 7, M // 2, M - 1]), protect)
    run_select(cc, weights, positions, lengths, M // 2, np.zeros(R, np.int64))      # every row protected
    run_select(cc, weights, positions, np.array([0, 1, M + 9, -4, M, M]), M // 3, np.full(R, 2 ** 30))


def test_select_rows_of_long_histories(cc):
    """Rows beyond what registers, and what LDS holds; strided inputs."""
    rng = np.random.default_rng(2)
    for M in (20000, 40001):
        weights = np.exp(2 * rng.standard_normal((2, M))).astype(np.float32)
        weights[1] = rng.integers(0, 50, M)
        positions = np.tile(np.arange(M, dtype=np.int32), (2, 1))
        run_select(cc, weights, positions, np.array([M, M - 7]), np.array([M // 2, M // 3]), np.array([M - 64, M - 64]))
    wide = torch.from_numpy(weights).cuda()
    pos = torch.from_numpy(positions).cuda()
    e = cc.select_rows(wide[:, 5:1005], pos[:, 5:1005], dev_i32([1000, 900]), 400, dev_i32([990, 890]))
    want = C.select(weights[:, 5:1005], positions[:, 5:1005], [1000, 900], [400, 400], [990, 890])
    for got, w in zip(e, want):
        assert (got.cpu().numpy() == w).all()


@pytest.mark.parametrize('M', [100, 3000, 9000, 33000])
def test_select_keeps_protected_rows_of_any_weight(cc, M):
    """As many protected rows as the budget, NaN and -inf among them, or all of them: each of them stays."""
    rng = np.random.default_rng(M)
    R, b = 4, M // 3
    weights = rng.standard_normal((R, M)).astype(np.float32)
    positions = np.stack([rng.permutation(M) for _ in range(R)]).astype(np.int32)
    kept = positions >= M - b
    weights[0, np.flatnonzero(kept[0])[:3]] = np.nan, -np.inf, -3.3e38
    weights[1, kept[1]] = np.nan
    weights[2, kept[2]] = -np.inf
    weights[3] = np.nan
    n = np.full(R, M, np.int32)
    e = run_select(cc, weights, positions, n, b, np.full(R, M - b))
    assert (np.sort(e.positions.cpu().numpy()[:, :b], 1) == np.arange(M - b, M)).all()


@pytest.mark.parametrize('width,block', [(128, 16), (256, 32), (512, 16), (1024, 48)])
def test_move_rows(cc, width, block):
    """Moved rows byte for byte, everything else untouched, on compact pages and on bf16 ones."""
    rng = np.random.default_rng(width)
    n = [90, 40, 0, 133]
    p = Pool(rng, n, width, block)
    M = 140
    weights = rng.random((4, M)).astype(np.float32)
    positions = np.tile(np.arange(M, dtype=np.int32), (4, 1))
    e = run_select(cc, weights, positions, np.array(n), 50, np.array([85, 0, 0, 130]))
    source, target = e.source.cpu().numpy(), e.target.cpu().numpy()
    cache, want = dev_u8(p.cache), p.cache.copy()
    for r in range(4):
        for s, t in zip(source[r], target[r]):
            if s >= 0:
                (a, x), (b, y) = (C.tile_of(want, int(C.slots_of(p.table[r], block, j + 1)[j])) for j in (s, t))
                for i, j in zip(C.addresses(width, x), C.addresses(width, y)):
                    b[j] = a[i]
    cc.move_rows(cache, dev_i32(p.table), e)
    assert (host_u8(cache) == want).all()
    cc.move_rows(cache, dev_i32(p.table), e)                    # sources are left as they are: again changes nothing
    assert (host_u8(cache) == want).all()
    bits = random_bits(rng, (len(p.cache), 1, block, 2 * width))
    pages, moved = dev_bf16(bits), bits.copy()
    for r in range(4):
        for s, t in zip(source[r], target[r]):
            if s >= 0:
                moved[p.table[r, t // block], 0, t % block] = bits[p.table[r, s // block], 0, s % block]
    cc.move_rows(pages, dev_i32(p.table), e)
    assert (pages.view(torch.int16).cpu().numpy().view(np.uint16) == moved).all()


def test_moves_through_bad_pages_are_skipped(cc):
    rng = np.random.default_rng(4)
    p = Pool(rng, [64], 128, 16, extra_cols=0)
    table = p.table.copy()
    table[0, 1], table[0, 2] = -1, len(p.cache)
    pairs = [[16, 40, 50, 63, 10 ** 6, 3, -1], [0, 1, 20, 2, 4, 10 ** 6, -1]]
    cache = dev_u8(p.cache)
    cc.move_rows(cache, dev_i32(table), cc.Eviction(None, None, None, dev_i32([pairs[0]]), dev_i32([pairs[1]])))
    got, rows = host_u8(cache), p.rows(0)
    after = C.load(got, C.slots_of(p.table[0], 16, 64))
    want = rows.copy()
    want[2] = rows[63]                                          # the only pair whose pages are both there
    assert (after == want).all()


# ---- together ------------------------------------------------------------------------------------------------------

def test_commit_attend_account_evict(cc, pkg):
    """A decoding loop: rows are committed step by step, every step attends and keeps account, then half of the rows go; what
    stays gives the attention over exactly those rows, and new rows go in behind them."""
    rng = np.random.default_rng(21)
    R, w, block, M, steps = 3, 256, 16, 96, 40
    cols = M // block
    table = rng.permutation(np.arange(1, 1 + R * cols)).reshape(R, cols).astype(np.int32)
    cache = torch.full((1 + R * cols, 1, 17 * w), 255, dtype=torch.uint8, device='cuda')
    account = torch.zeros(R, M, device='cuda')
    positions = torch.full((R, M), -1, dtype=torch.int32, device='cuda')
    lengths = np.zeros(R, np.int32)
    kept = [[] for _ in range(R)]                               # bf16 rows by slot order, on the host
    qsl, d_table = dev_i32(np.arange(R + 1)), dev_i32(table)
    want_w = np.zeros((R, M))
    for step in range(steps):
        rows = latents(rng, (R, 2 * w))
        bits = dev_bf16(rows)
        slots = [int(C.slots_of(table[r], block, lengths[r] + 1)[-1]) for r in range(R)]
        cc.store_rows(bits[:, :w], bits[:, w:], dev_i64(slots), cache)
        for r in range(R):
            kept[r].append(C.values(*C.quantise(bf16.to_f32(rows[r].reshape(2, w)))).reshape(-1))
            positions[r, lengths[r]] = step
        lengths += 1
        q = random_bits(rng, (R, 16, w))
        ctx = dev_i32(lengths)
        o, lse = cc.history_attention(dev_bf16(q), cache, d_table, ctx, SCALE, M)
        check_attention(host_f32(o), host_f32(lse), bf16.to_f32(q), lambda t: np.stack(kept[t]), lengths)
        cc.attention_weights(dev_bf16(q), cache, d_table, qsl, ctx, lse, SCALE, account)
        if step == 29:
            before = account.cpu().numpy()
            e = cc.select_rows(account, positions, ctx, 15, dev_i32([step - 3] * R))
            cc.move_rows(cache, d_table, e)
            want = C.select(before, positions.cpu().numpy(), lengths, [15] * R, [step - 3] * R)
            assert all((a.cpu().numpy() == b).all() for a, b in zip(e, want))
            for r in range(R):
                place = positions[r].cpu().numpy()
                at = [int(np.where(place == x)[0][0]) for x in e.positions[r, :15].cpu().numpy()]
                kept[r] = [kept[r][j] for j in at]
            account, positions, lengths = e.weights, e.positions, e.lengths.cpu().numpy().copy()
            assert (lengths == 15).all()


def layer_step(pkg, ops, rng, contexts, chunk, R_cols, w, ctx_kwargs=None):
    """A StepContext of requests with `contexts` cached tokens and `chunk` new ones each, and the tensors of a layer."""
    B, W = len(contexts), 32
    T, H, D = B * chunk, 16, 128
    qsl = np.arange(0, T + 1, chunk)
    seq = np.asarray(contexts) + chunk
    positions = np.concatenate([np.arange(c, c + chunk) for c in contexts])
    table = pkg.s6_layer.latent_rope_table(2048, pkg.s6_layer.latent_inv_freq(D, 1e4), w, torch.bfloat16).cuda()
    ctx = pkg.s6_layer.StepContext(dev_i64(positions), dev_i32(qsl), dev_i32(seq), chunk, T, {w: table}, SCALE,
                                   ops.select_backends(), ops.S6Workspace(H, w, 4096), 4, window=W, max_seqlen_k=int(seq.max()))
    return ctx, T


@pytest.mark.parametrize('chunk', [1, 3, 20])
@pytest.mark.parametrize('w', [256, 512])
def test_attend_over_a_compact_cache(cc, pkg, ops, w, chunk):
    """s6_layer.attend over a compact cache equals attend over the bf16 cache that holds the same values, with and without
    an account: one kind of rounding step (the weights', the history output's, the merged output's) of 2^-8 on each side."""
    rng = np.random.default_rng(w + chunk)
    contexts = [300, 90, 20, 33]
    H, D, block = 16, 128, 16
    ctx, T = layer_step(pkg, ops, rng, contexts, chunk, None, w)
    p = Pool(rng, [c + chunk for c in contexts], w, block)
    pages = len(p.cache)
    every = np.nan_to_num(C.load(p.cache, np.arange(pages * block)))
    plain = torch.from_numpy(every.reshape(pages, 1, block, 2 * w)).to(torch.bfloat16).cuda()
    exact = dev_bf16(random_bits(rng, (pages, H, block, 2 * D)))
    q_lat = dev_bf16(random_bits(rng, (T, H, w), 1.4 * math.sqrt(128 / w)))
    q_rope, k_rope, v = (dev_bf16(random_bits(rng, (T, H, D))) for _ in range(3))
    B = dev_bf16(random_bits(rng, (H, w, D), 1 / math.sqrt(w)))
    layer = FakeLatentLayer(B, B, [B], [B])
    layer.rank1 = layer.rank = w
    table = dev_i32(p.table)
    pos = dev_i64(np.concatenate([np.arange(c, c + chunk) for c in contexts]))
    for t in range(T):   # the adapter writes the chunk's own exact rows before it attends
        r, j = t // chunk, int(pos[t])
        page, x = int(p.table[r, j // block]), j % block
        exact[page, :, x, :D], exact[page, :, x, D:] = k_rope[t], v[t]
    args = lambda c: (layer, 0, q_lat, q_rope, k_rope, v, c, table, None, None, ctx, (exact, table))
    want = pkg.s6_layer.attend(*args(plain)).float()
    M = 310
    a1, a2 = torch.zeros(4, M, device='cuda'), torch.zeros(4, M, device='cuda')
    outs = [pkg.s6_layer.attend(*args(dev_u8(p.cache))), pkg.s6_layer.attend(*args(dev_u8(p.cache)), weights=a1),
            pkg.s6_layer.attend(*args(plain), weights=a2)]
    for got in outs:
        # |o| is at most the largest of a few hundred values of size about 1, each off by at most 4 roundings of 2^-8
        assert (got.float() - want).abs().max() <= 4 * HALF * want.abs().max()
        assert (got.float() - want).norm() <= 2 * HALF * want.norm()
    assert torch.allclose(a1, a2, rtol=2.0 ** -10, atol=1e-6)   # lse and scores differ by fp32 sums alone
    total = a1.sum(1).cpu().numpy()
    # the window has its share, and all of it where a request has no row behind it
    assert ((total > 0) == (np.array(contexts) > 32)).all() and (total < 16 * chunk).all()
    for r, c in enumerate(contexts):
        assert (a1[r, max(c - 32, 0):] == 0).all()


def test_attend_after_an_eviction(cc, pkg, ops):
    """A layer with an exact window: the rows behind the window are evicted by the account that attend keeps, the window's rows
    follow them, and the next step attends to what is left, as over a bf16 cache of the same rows."""
    rng = np.random.default_rng(5)
    contexts, w, block, W, b, H, D = [300, 200, 150, 120], 512, 16, 32, 40, 16, 128
    ctx, T = layer_step(pkg, ops, rng, contexts, 1, None, w)
    p = Pool(rng, [c + 1 for c in contexts], w, block)
    cache, table = dev_u8(p.cache), dev_i32(p.table)
    exact = dev_bf16(random_bits(rng, (len(p.cache), H, block, 2 * D)))
    q_lat = dev_bf16(random_bits(rng, (T, H, w), 0.7))
    q_rope, k_rope, v = (dev_bf16(random_bits(rng, (T, H, D))) for _ in range(3))
    B = dev_bf16(random_bits(rng, (H, w, D), 1 / math.sqrt(w)))
    layer = FakeLatentLayer(B, B, [B], [B])
    layer.rank1 = layer.rank = w
    account = torch.zeros(4, 300, device='cuda')
    step = lambda c, x, **kw: pkg.s6_layer.attend(layer, 0, q_lat, q_rope, k_rope, v, c, table, None, None, x, (exact, table), **kw)
    step(cache, ctx, weights=account)
    behind = ctx.ctx_latent.clone()
    assert behind.tolist() == [c - W for c in contexts]
    positions = torch.arange(300, dtype=torch.int32, device='cuda').repeat(4, 1)
    e = cc.select_rows(account, positions, behind, b, behind)          # nothing protected
    cc.move_rows(cache, table, e)
    i = torch.arange(W, dtype=torch.int32, device='cuda')
    cc.move_rows(cache, table, cc.Eviction(None, None, None, behind[:, None] + i, e.lengths[:, None] + i))
    assert e.lengths.tolist() == [b] * 4
    got, plain = host_u8(cache), np.zeros((len(p.cache), 1, block, 2 * w), np.float32)
    for r, c in enumerate(contexts):
        kept = np.concatenate((e.positions[r, :b].cpu().numpy(), np.arange(c - W, c)))
        assert len(set(kept)) == b + W and kept[:b].max() < c - W
        slots = C.slots_of(p.table[r], block, b + W)
        assert (C.load(got, slots) == p.rows(r)[kept]).all()
        plain[slots // block, 0, slots % block] = p.rows(r)[kept]
    steps = []
    for _ in range(2):
        x, _ = layer_step(pkg, ops, rng, contexts, 1, None, w)
        x.ctx_latent.copy_(e.lengths)
        steps.append(x)
    want = step(torch.from_numpy(plain).to(torch.bfloat16).cuda(), steps[0]).float()
    out = step(cache, steps[1]).float()
    assert (out - want).abs().max() <= 4 * HALF * want.abs().max() and (out - want).norm() <= 2 * HALF * want.norm()


def test_write_commit_into_a_compact_cache(cc, pkg, ops):
    """write_commit and store_rows put the same bytes into a compact cache as the quantised rows of the bf16 path."""
    rng = np.random.default_rng(31)
    w, hidden, chunk, contexts = 256, 512, 5, [10, 40]
    ctx, T = layer_step(pkg, ops, rng, contexts, chunk, None, w)
    lin = torch.nn.Linear(hidden, 2 * w, bias=False, device='cuda', dtype=torch.bfloat16)
    layer = FakeLatentLayer(torch.empty(16, 128, w), None, [torch.empty(16, 128, w)], None)
    layer.cand1, layer.rank1 = lin, w
    h = dev_bf16(random_bits(rng, (T, hidden)))
    table = np.arange(1, 9, dtype=np.int32).reshape(2, 4)
    plain = torch.zeros(9, 1, 16, 2 * w, dtype=torch.bfloat16, device='cuda')
    compact = torch.zeros(cc.cache_shape(9, 16, w), dtype=torch.uint8, device='cuda')
    with torch.no_grad():
        pkg.s6_layer.write_commit(layer, 0, h, None, ctx, plain, dev_i32(table))
        pkg.s6_layer.write_commit(layer, 0, h, None, ctx, compact, dev_i32(table))
    slots = np.concatenate([C.slots_of(table[r], 16, c + chunk)[c:] for r, c in enumerate(contexts)])
    rows = host_f32(plain.view(-1, 2 * w))[slots]
    want = np.zeros(cc.cache_shape(9, 16, w), np.uint8)
    C.store(want, rows[:, :w], rows[:, w:], slots)
    assert (host_u8(compact) == want).all()
    again = torch.zeros_like(compact)
    bits = plain.view(-1, 2 * w)[torch.from_numpy(slots).cuda()]
    pkg.s6_layer.store_rows(bits[:, :w], bits[:, w:], dev_i64(slots), again)
    assert torch.equal(again, compact)


def test_captured_step(cc):
    """A captured step (commit, attention, account, eviction) replayed with new inputs, eager work and synchronizations
    between the replays; every replay equals the eager calls."""
    rng = np.random.default_rng(41)
    w, n = 256, [150, 60]
    p = Pool(rng, n, w, 16)
    cache, table, ctx, qsl = dev_u8(p.cache), dev_i32(p.table), dev_i32(n), dev_i32([0, 1, 2])
    q = torch.zeros(2, 16, w, dtype=torch.bfloat16, device='cuda')
    rows = torch.zeros(2, 2 * w, dtype=torch.bfloat16, device='cuda')
    slots = dev_i64([int(C.slots_of(p.table[r], 16, n[r])[-1]) for r in range(2)])
    account = torch.zeros(2, 150, device='cuda')
    positions = torch.arange(150, dtype=torch.int32, device='cuda').repeat(2, 1)

    def step():
        cc.store_rows(rows[:, :w], rows[:, w:], slots, cache)
        o, lse = cc.history_attention(q, cache, table, ctx, SCALE, 150)
        cc.attention_weights(q, cache, table, qsl, ctx, lse, SCALE, account)
        e = cc.select_rows(account, positions, ctx, 50, dev_protect)
        cc.move_rows(cache, table, e)
        return (o, lse, *e)

    dev_protect = dev_i32([140, 50])
    first = cache.clone()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    for trial in range(3):
        q.copy_(dev_bf16(random_bits(rng, (2, 16, w))))
        rows.copy_(dev_bf16(latents(rng, (2, 2 * w))))
        cache.copy_(first)
        account.zero_()
        graph.replay()
        torch.cuda.synchronize()
        got = [x.clone() for x in out] + [cache.clone(), account.clone()]
        cache.copy_(first)
        account.zero_()
        want = list(step()) + [cache, account]
        torch.cuda.synchronize()
        for a, b in zip(got, want):
            assert torch.equal(a, b), trial


def test_another_stream(cc):
    rng = np.random.default_rng(43)
    p = Pool(rng, [500], 512, 16)
    cache, table, q = dev_u8(p.cache), dev_i32(p.table), dev_bf16(random_bits(rng, (1, 16, 512)))
    want = cc.history_attention(q, cache, table, dev_i32([500]), SCALE, 500)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = cc.history_attention(q, cache, table, dev_i32([500]), SCALE, 500)
    side.synchronize()
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


def test_refusals(cc):
    z = lambda *s, dtype=torch.bfloat16: torch.zeros(*s, dtype=dtype, device='cuda')
    i32 = lambda *s: z(*s, dtype=torch.int32)
    i64 = lambda *s: z(*s, dtype=torch.int64)
    cache, table, q, rows = z(4, 1, 17 * 256, dtype=torch.uint8), i32(2, 3), z(2, 16, 256), z(2, 256)
    bf = z(4, 1, 16, 512)
    bad = [
        (lambda: cc.cache_shape(4, 24, 256), 'block size'),
        (lambda: cc.cache_shape(4, 16, 384), 'width'),
        (lambda: cc.store_rows(rows.float(), rows, i64(2), cache), 'bfloat16'),
        (lambda: cc.store_rows(rows, z(2, 128), i64(2), cache), 'alike'),
        (lambda: cc.store_rows(rows, rows, i64(3), cache), 'slots'),
        (lambda: cc.store_rows(rows, rows, i32(2), cache), 'slots'),
        (lambda: cc.store_rows(rows, rows, i64(2), cache.float()), 'uint8'),
        (lambda: cc.store_rows(z(2, 512), z(2, 512), i64(2), cache), 'compact cache'),
        (lambda: cc.load_rows(cache, table, i32(3), 8), 'rows'),
        (lambda: cc.load_rows(cache, table, i32(2), 8, out=z(2, 7, 512)), 'out'),
        (lambda: cc.load_rows(cache[:, :, :256], table, i32(2), 8), 'compact cache'),
        (lambda: cc.load_rows(z(4, 17 * 256, 2, dtype=torch.uint8).transpose(1, 2), table, i32(2), 8), 'contiguous'),
        (lambda: cc.history_attention(z(2, 8, 256), cache, table, i32(2), 1.0, 8), '16'),
        (lambda: cc.history_attention(z(2, 16, 512), cache, table, i32(2), 1.0, 8), 'compact cache'),
        (lambda: cc.history_attention(q, cache, table[:1], i32(2), 1.0, 8), 'block_table'),
        (lambda: cc.history_attention(q, cache, table, i32(3), 1.0, 8), 'ctx'),
        (lambda: cc.history_attention(q, cache, table, i64(2), 1.0, 8), 'ctx'),
        (lambda: cc.history_attention(q, cache, table, i32(2), 1.0, 8, token_requests=i64(1)), 'token_requests'),
        (lambda: cc.history_attention(q, cache, table, i32(2), 1.0, 8, num_kv_splits=0), 'num_kv_splits'),
        (lambda: cc.history_attention(q, cache, table, i32(2), 1.0, 8, num_kv_splits=2, plan=i32(3)), 'plan'),
        (lambda: cc.history_attention(z(2, 16, 260)[:, :, 2:258], cache, table, i32(2), 1.0, 8), 'aligned'),
        (lambda: cc.attention_weights(q, cache, table, i32(3), i32(2), z(16, 3).float(), 1.0, z(2, 9).float()), 'lse'),
        (lambda: cc.attention_weights(q, cache, table, i32(3), i32(2), z(16, 2).float(), 1.0, z(3, 9).float()), 'weights'),
        (lambda: cc.attention_weights(q, cache, table, i32(3), i32(2), z(16, 2).float(), 1.0, z(2, 9)), 'weights'),
        (lambda: cc.attention_weights(q, z(4, 2, 16, 512), table, i32(3), i32(2), z(16, 2).float(), 1.0, z(2, 9).float()),
         'latent cache'),
        (lambda: cc.select_rows(z(2, 9), i32(2, 9), i32(2), 4, i32(2)), 'weights'),
        (lambda: cc.select_rows(z(2, 9).float(), i32(2, 8), i32(2), 4, i32(2)), 'positions'),
        (lambda: cc.select_rows(z(2, 9).float(), i32(2, 9), i32(3), 4, i32(2)), 'lengths'),
        (lambda: cc.select_rows(z(2, 9).float(), i32(2, 9), i32(2), -1, i32(2)), 'budget'),
        (lambda: cc.select_rows(z(2, 9).float(), i32(2, 9), i32(2), i32(3), i32(2)), 'budget'),
        (lambda: cc.move_rows(bf, table, cc.Eviction(None, None, None, i32(2, 4), i32(2, 5))), 'target'),
        (lambda: cc.move_rows(bf, table, cc.Eviction(None, None, None, i32(3, 4), i32(3, 4))), 'block_table'),
        (lambda: cc.move_rows(bf.float(), table, cc.Eviction(None, None, None, i32(2, 4), i32(2, 4))), 'bfloat16'),
    ]
    for call, match in bad:
        with pytest.raises(ValueError, match=match):
            call()
    with pytest.raises(RuntimeError, match='S6Workspace'):
        cc.history_partials(q, cache, table, i32(2), 1.0, 2, None)
    small = type('W', (), {'attn_logits': lambda self, *a: z(10).float()})()
    with pytest.raises(RuntimeError, match='overflow'):
        cc.history_attention(q, cache, table, i32(2), 1.0, 8, num_kv_splits=2, workspace=small)


def test_nothing_to_do(cc):
    """No tokens, no requests, no rows."""
    z = lambda *s, dtype=torch.int32: torch.zeros(*s, dtype=dtype, device='cuda')
    cache, q = z(4, 1, 17 * 128, dtype=torch.uint8), z(0, 16, 128, dtype=torch.bfloat16)
    o, lse = cc.history_attention(q, cache, z(0, 3), z(0), 1.0, 0)
    assert o.shape == (0, 16, 128) and lse.shape == (16, 0)
    assert cc.load_rows(cache, z(0, 3), z(0), 5).shape == (0, 5, 256)
    assert cc.load_rows(cache, z(2, 3), z(2), 0).shape == (2, 0, 256)
    account = torch.ones(2, 7, device='cuda')
    cc.attention_weights(q, cache, z(2, 3), z(3), z(0), torch.zeros(16, 0, device='cuda'), 1.0, account)
    assert (account == 1).all()
    e = cc.select_rows(torch.ones(2, 0, device='cuda'), z(2, 0), z(2), 4, z(2))
    assert e.lengths.tolist() == [0, 0] and e.source.shape == (2, 0)
    cc.move_rows(cache, z(2, 3), e)
